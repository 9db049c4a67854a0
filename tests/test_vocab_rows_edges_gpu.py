"""Operators over rows of logits where they can go wrong: fills of a mask, loss factors, head-level gradients, rows whose
entries cover all that lives, shards of the vocabulary.  Tolerances are those derived in test_vocab_rows_gpu.py, or stated
at the test."""

import math

import pytest
import torch

from tests import vocab_oracle as oracle
from tests.test_vocab_rows_gpu import (DEV, ROUND, TINY, TYPES, _check_distill, _check_grad, _check_logp, _check_top,
                                       _close, _logits, _ops, _teacher)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ masks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", [-1e9, -1e10, -3e12, -1e20, -1e29])
@pytest.mark.parametrize("vocab", [777, 100003])
def test_finite_masks(dtype, fill, vocab):
    """Masks that are neither infinite nor the type's lowest value, in rows where whole threads see nothing else."""
    x = _logits(5, vocab, dtype, seed=vocab)
    x[0, 100:] = fill
    x[1, : vocab - 30] = fill
    x[2] = fill
    x[2, vocab // 2] = 1.5
    x[3, ::2] = fill
    ids, logq = _teacher(5, vocab, 6)
    live = torch.tensor([[3, 70], [vocab - 1, vocab - 9], [vocab // 2, vocab // 2], [1, 11], [0, 5]], device=DEV)
    ids[:, :2] = live
    ids[2, 1] = -1
    ids[:4, 2:] = -1                               # (a given token that the student rules out is another test's)
    logq = torch.where(ids >= 0, logq - 1.0, logq)
    for temp in (1.0, 0.7):
        xg = x.detach().requires_grad_()
        r = _ops().token_logprobs(xg, live, temp, top_k=4)
        _check_logp(r, x, live, temp)
        _check_top(_ops().token_logprobs(x[3:], None, temp, top_k=9), x[3:], temp, 9)
        d, dh = torch.randn(5, 2, device=DEV), torch.randn(5, device=DEV)
        (got,) = torch.autograd.grad((r.logp, r.entropy), xg, (d, dh))
        size = ((d.abs().sum(1) + 32 * dh.abs()) / temp)[:, None].double()
        _check_grad(got, oracle.token_grad(x, live, temp, d, dh), size, dtype)
        _check_distill(x, ids, logq, tail=False, temp=temp)
        _check_distill(x[[0, 1, 3, 4]], ids[[0, 1, 3, 4]], logq[[0, 1, 3, 4]], tail=True, temp=temp)


@pytest.mark.parametrize("fill", [-1e10, -1e15, -1e25])
def test_rows_of_finite_masks_carry_nothing(fill):
    for vocab in (300, 70001):
        x = torch.full((2, vocab), fill, device=DEV).requires_grad_()
        r = _ops().token_logprobs(x, torch.tensor([1, 2], device=DEV), top_k=3)
        assert bool((r.logp == -math.inf).all()) and r.entropy.tolist() == [0.0, 0.0]
        assert r.top_ids.tolist() == [[0, 1, 2]] * 2 and bool((r.top_logp == -math.inf).all())
        (g,) = torch.autograd.grad((r.logp, r.entropy), x, (torch.ones(2, device=DEV), torch.ones(2, device=DEV)))
        assert not bool(g.any())
        _, rows = _ops().topk_distill_loss(x.detach(), torch.zeros(2, 1, dtype=torch.long, device=DEV),
                                           torch.full((2, 1), -0.5, device=DEV), denom=1.0)
        assert rows.tolist() == [math.inf] * 2


def test_logits_beyond_the_range_are_nan():
    """x / T above 2^31 ln 2 has no FP32 reference near enough: NaN, as for infinite logits, in that row alone."""
    for vocab in (300, 70001):
        x = _logits(3, vocab, torch.float32)
        x[1, 40] = 3e10
        xg = x.clone().requires_grad_()
        tokens = torch.tensor([1, 40, 3], device=DEV)
        r = _ops().token_logprobs(xg, tokens, top_k=4)
        assert torch.isnan(r.logp).tolist() == [False, True, False] == torch.isnan(r.entropy).tolist()
        assert torch.equal(r.top_ids, oracle.top(x, 4))
        (g,) = torch.autograd.grad(r.logp.sum(), xg)
        assert bool(torch.isnan(g[1]).all()) and bool(torch.isfinite(g[::2]).all())


# ------------------------------------------------------------------------------------------------ heads
def _head(U=200, H=128, V=1000, K=8, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = (torch.randn(U, H, device=DEV, generator=g) * 0.5).to(dtype)
    W = (torch.randn(V, H, device=DEV, generator=g) * 0.2).to(dtype)
    ids, logq = _teacher(U, V, K, seed)
    w = 0.2 + torch.rand(U, device=DEV, generator=g)
    return h, W, ids, logq, w


def test_head_loss_without_gradient_leaves_main_grad_alone():
    ops = _ops()
    h, W, ids, logq, w = _head()
    W.requires_grad_()
    W.main_grad = torch.zeros(W.shape, device=DEV)
    with torch.no_grad():
        loss, rows = ops.fused_lm_head_topk_distill(h, W, ids, logq, denom=200.0, weights=w, chunk_rows=64)
    assert not loss.requires_grad and not bool(W.main_grad.any())
    want, _ = oracle.distill(h.float() @ W.detach().float().t(), ids, logq, 1.0, True)
    _close(rows, want, 5e-2, 1e-2, "rows")


@pytest.mark.parametrize("main", [True, False])
@pytest.mark.parametrize("announced,factor", [(1.0, 0.5), (1.0, 1.0), (49.0, 7.0)])
def test_head_gradients_agree_for_any_loss_factor(main, announced, factor):
    """Tolerances of BF16 logits and their BF16 gradients, as at the other test of the head."""
    h, W, ids, logq, w = _head()
    h.requires_grad_()
    W.requires_grad_()
    if main:
        W.main_grad = torch.full(W.shape, 2.0, device=DEV)
    loss, _ = _ops().fused_lm_head_topk_distill(h, W, ids, logq, denom=200.0, weights=w, chunk_rows=64,
                                                grad_scale=announced)
    assert not main or bool((W.main_grad == 2.0).all())
    (loss * factor).backward()
    hd, Wd = h.detach().double(), W.detach().double()
    _, gx = oracle.distill(hd @ Wd.t(), ids, logq, 1.0, True)
    gx = gx * w.double()[:, None] * factor / 200.0
    dh, dw = gx @ Wd, gx.t() @ hd
    got = W.main_grad - 2.0 if main else W.grad
    _close(h.grad, dh, 2e-2 * float(dh.abs().max()), 5e-2, "dh")
    _close(got, dw, 2e-2 * float(dw.abs().max()), 5e-2, "dW")


# ---------------------------------------------------------------------------------------- loss factors
@pytest.mark.parametrize("rows,vocab", [(64, 1024), (5, 30011), (400, 30000)])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("announced,factor", [(1.0, 16384.0), (49.0, 98304.0), (16384.0, 16384.0)])
def test_unannounced_loss_scale_in_fp16(rows, vocab, tail, announced, factor):
    """A gradient that underflows unscaled is rounded once, after the scale; the rows stay what they were."""
    x = _logits(rows, vocab, torch.float16).requires_grad_()
    ids, logq = _teacher(rows, vocab, 8)
    w = 0.1 + torch.rand(rows, device=DEV)
    w[0] = 0.0
    loss, kl = _ops().topk_distill_loss(x, ids, logq, denom=4096.0, weights=w, grad_scale=announced, tail=tail)
    keep = kl.clone()
    (got,) = torch.autograd.grad(loss * factor, x, retain_graph=True)
    _, want = oracle.distill(x.detach(), ids, logq, 1.0, tail)
    f = w.double()[:, None] * factor / 4096.0
    _check_grad(got, want * f, 2 * f, torch.float16)
    assert torch.equal(kl, keep)
    with pytest.raises(RuntimeError, match="already taken"):
        torch.autograd.grad(loss, x)


@pytest.mark.parametrize("main", [True, False])
@pytest.mark.parametrize("temp", [1.0, "rows"])
def test_head_unannounced_loss_scale_in_fp16(main, temp):
    """FP16 logits (2^-11 of their size, below 8) and FP16 products of gradients that would underflow unscaled."""
    h, W, ids, logq, w = _head(dtype=torch.float16)
    h.requires_grad_()
    W.requires_grad_()
    if main:
        W.main_grad = torch.zeros(W.shape, device=DEV)
    t = 0.8 + torch.rand(200, device=DEV) if temp == "rows" else temp
    scale = 2.0 ** 20
    loss, _ = _ops().fused_lm_head_topk_distill(h, W, ids, logq, denom=2.0 ** 25, weights=w, temperature=t, chunk_rows=64)
    (loss * scale).backward()
    hd, Wd = h.detach().double(), W.detach().double()
    _, gx = oracle.distill(hd @ Wd.t(), ids, logq, t, True)
    gx = gx * w.double()[:, None] * scale / 2.0 ** 25
    dh, dw = gx @ Wd, gx.t() @ hd
    got = W.main_grad if main else W.grad
    assert float((h.grad - dh).abs().max()) <= 2.0 ** -6 * float(dh.abs().max())
    assert float((got - dw).abs().max()) <= 2.0 ** -6 * float(dw.abs().max())


# -------------------------------------------------------------------------------- no second derivative
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_second_derivatives_and_forward_mode_are_refused(dtype):
    from torch.autograd import forward_ad

    ops = _ops()
    x = _logits(3, 50, dtype).requires_grad_()
    tokens = torch.tensor([1, 2, 3], device=DEV)
    ids, logq = _teacher(3, 50, 4)
    r = ops.token_logprobs(x, tokens)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x, create_graph=True)
    loss, _ = ops.topk_distill_loss(x, ids, logq, denom=3.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, x, create_graph=True, retain_graph=True)
    assert bool(torch.autograd.grad(loss, x)[0].any())          # (the refusal took nothing away)
    h, W, ids, logq, _ = _head()
    loss, _ = ops.fused_lm_head_topk_distill(h.requires_grad_(), W, ids, logq, denom=200.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, h, create_graph=True)
    with forward_ad.dual_level():
        for grad in (False, True):
            y = forward_ad.make_dual(x.detach().requires_grad_(grad), torch.randn_like(x))
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.token_logprobs(y, tokens)
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.topk_distill_loss(y, ids[:3] % 50, logq[:3], denom=3.0)


# --------------------------------------------------------------------------- teachers that cover all that lives
@pytest.mark.parametrize("vocab", [120, 2000, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_teacher_of_all_live_tokens_is_finite(vocab, dtype):
    """The operator's own alternatives of masked rows, to a student under the same mask: the KL of the live tokens."""
    from tests.test_vocab_rows_edges_cpu import _covered, _kl_of_live

    t, x = (v.to(dtype) for v in _covered(rows=32, vocab=vocab, device=DEV))
    ops = _ops()
    for temp in (1.0, 0.6):
        teacher = ops.token_logprobs(t, None, temp, top_k=64)
        xg = x.detach().requires_grad_()
        loss, rows = ops.topk_distill_loss(xg, teacher.top_ids, teacher.top_logp, denom=1.0, temperature=temp)
        want, grad = _kl_of_live(t, x, temp)
        _close(rows, want, 8e-6, 1e-6, "rows")                # (2e-6 of every log-prob of the teacher besides)
        assert bool(torch.isfinite(loss))
        _check_grad(torch.autograd.grad(loss, xg)[0], grad, torch.full((32, 1), 2.0 / temp, device=DEV).double(), dtype)
        _, rows = ops.topk_distill_loss(x, teacher.top_ids, teacher.top_logp - 1e-3, denom=1.0, temperature=temp)
        assert bool((rows == math.inf).all())


def test_teacher_of_all_live_tokens_in_shards():
    from bridge_b200.ops._ext import kernels
    from tests.test_vocab_rows_edges_cpu import _covered, _kl_of_live

    m = kernels()
    t, x = _covered(rows=32, vocab=900, device=DEV)
    teacher = _ops().token_logprobs(t, top_k=64)
    stats, xc = m.distill_open(x, teacher.top_ids, teacher.top_logp, None, None, 1.0, 0, 900)
    rows, coef, fix = m.distill_finish(stats, xc, teacher.top_ids, teacher.top_logp, None, None, 1.0, 1.0, True, 900)
    want, grad = _kl_of_live(t, x)
    _close(rows, want, 1e-5, 2e-6, "rows")
    got = m.distill_grad(x, teacher.top_ids, coef, fix, None, 1.0, 0, 900, False)
    _check_grad(got, grad, torch.full((32, 1), 4.0, device=DEV).double(), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_announced_scales_leave_the_gradient_alone(dtype):
    """The gradient of a loss scaled as announced is the forward's own, bit for bit and without a write, whatever the
    announced number: also where a reciprocal's product would not give exactly 1."""
    x = _logits(4, 600, dtype).requires_grad_()
    ids, logq = _teacher(4, 600, 5)
    from bridge_b200.ops._ext import kernels

    for scale in [*range(1, 200), 1.1, 3e-3, 12345.678]:
        own = x.detach().clone()
        kernels().distill_rows_inplace(own, ids, logq, None, None, 1.0, scale / 7.0, True, True)
        loss, _ = _ops().topk_distill_loss(x, ids, logq, denom=7.0, grad_scale=scale)
        (got,) = torch.autograd.grad(loss, x, torch.tensor(scale, device=DEV))
        assert torch.equal(got, own), scale


# ------------------------------------------------------------------------------------ vocabularies in shards
def _ranks(monkeypatch, n, work):
    """``work(rank, group)`` on ``n`` threads of this process, with collectives between the threads on the host."""
    import threading

    from bridge_b200.ops import distill, token_logprob

    barrier, slots, me = threading.Barrier(n, timeout=60), [None] * n, threading.local()

    def everyone(t):
        slots[me.rank] = t.clone()
        barrier.wait()
        got = list(slots)
        barrier.wait()
        return got

    class Dist:
        ReduceOp = torch.distributed.ReduceOp

        @staticmethod
        def get_world_size(group):
            return n

        @staticmethod
        def all_reduce(t, op=torch.distributed.ReduceOp.SUM, group=None):
            got = torch.stack(everyone(t))
            t.copy_(got.amax(0) if op == torch.distributed.ReduceOp.MAX else got.sum(0))

        @staticmethod
        def all_gather(out, t, group=None):
            for o, v in zip(out, everyone(t)):
                o.copy_(v)

    for module in (distill, token_logprob):
        monkeypatch.setattr(module, "dist", Dist)
    out, failed = [None] * n, []

    def run(rank):
        me.rank = rank
        try:
            out[rank] = work(rank, "threads")
        except BaseException as exc:  # noqa: BLE001 - raised again below
            failed.append(exc)
            barrier.abort()

    threads = [threading.Thread(target=run, args=(r,)) for r in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temp", [0.9, "rows"])
def test_scores_in_shards(monkeypatch, dtype, temp):
    """The whole call on every rank, at the whole row's tolerance, with logits far from 0."""
    rows, part, n = 40, 1501, 3
    vocab = n * part
    x = _logits(rows, vocab, dtype) + 60.0
    x[4, part:2 * part] = -math.inf
    x[5] = -math.inf
    tokens = torch.randint(0, vocab, (rows, 2), device=DEV)
    tokens[0, 1] = -1
    t = 0.5 + torch.rand(rows, device=DEV) if temp == "rows" else temp
    d, dh = torch.randn(rows, 2, device=DEV), torch.randn(rows, device=DEV)

    def work(rank, group):
        mine = x[:, rank * part:(rank + 1) * part].clone().requires_grad_()
        r = _ops().token_logprobs(mine, tokens, t, top_k=20, vocab_start=rank * part, tp_group=group)
        return r, torch.autograd.grad((r.logp, r.entropy), mine, (d, dh))[0]

    got = _ranks(monkeypatch, n, work)
    for r, _ in got:
        _check_logp(r, x, tokens, t)
        _check_top(r, x, t, 20)
        assert r.logp.dtype == r.entropy.dtype == r.top_logp.dtype == torch.float32
    size = ((d.abs().sum(1) + 32 * dh.abs()) / t)[:, None].double()
    _check_grad(torch.cat([g for _, g in got], 1), oracle.token_grad(x, tokens, t, d, dh), size, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_in_shards(monkeypatch, dtype, tail):
    """Loss and gradient on every rank, under a loss scale that was not announced; tolerances of the open form's test."""
    rows, part, n = 20, 1001, 3
    x = _logits(rows, n * part, dtype)
    ids, logq = _teacher(rows, n * part, 9)
    ids[1, 4:] = -1
    w = torch.rand(rows, device=DEV) + 0.1

    def work(rank, group):
        mine = x[:, rank * part:(rank + 1) * part].clone().requires_grad_()
        loss, kl = _ops().topk_distill_loss(mine, ids, logq, denom=4096.0, weights=w, temperature=0.9, tail=tail,
                                            vocab_start=rank * part, tp_group=group)
        return loss.detach(), kl, torch.autograd.grad(loss * 16384.0, mine)[0]

    got = _ranks(monkeypatch, n, work)
    kl_want, g_want = oracle.distill(x, ids, logq, 0.9, tail)
    for loss, kl, _ in got:
        _close(kl, kl_want, 1e-5, 2e-6, "rows")
        _close(loss, (kl_want * w.double()).sum() / 4096.0, 1e-5, 2e-6, "loss")
    f = (w.double() * 4.0)[:, None]
    _check_grad(torch.cat([g for *_, g in got], 1), g_want * f, 4 * f, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads_in_shards(monkeypatch, dtype):
    """Teacher alternatives and the student's loss through heads in shards against the whole head on one rank."""
    ops = _ops()
    h, W, *_ = _head(V=1200, dtype=dtype)
    w = 0.2 + torch.rand(200, device=DEV)
    whole = ops.fused_lm_head_token_logprobs(h, W, top_k=8, chunk_rows=64)

    def student(Wr, group=None, start=0):
        hr = h.clone().requires_grad_()
        Wr = Wr.clone().requires_grad_()
        Wr.main_grad = torch.zeros(Wr.shape, device=DEV)
        loss, kl = ops.fused_lm_head_topk_distill(hr, Wr, whole.top_ids, whole.top_logp, denom=200.0, weights=w,
                                                  chunk_rows=64, vocab_start=start, tp_group=group)
        (loss * 0.5).backward()
        return loss.detach(), kl, hr.grad, Wr.main_grad

    Ws = (W.float() + 0.05 * torch.randn(W.shape, device=DEV)).to(dtype)
    loss, kl, dh, dw = student(Ws)

    def work(rank, group):
        at = slice(rank * 400, (rank + 1) * 400)
        r = ops.fused_lm_head_token_logprobs(h, W[at], top_k=8, chunk_rows=64, vocab_start=rank * 400, tp_group=group)
        return r, student(Ws[at], group, rank * 400)

    got = _ranks(monkeypatch, 3, work)
    for r, s in got:
        assert torch.equal(r.top_ids, whole.top_ids)
        _close(r.top_logp, whole.top_logp, 4e-6, 1e-6, "teacher")
        _close(s[0], loss, 1e-5, 4e-6, "loss")
        _close(s[1], kl, 1e-5, 4e-6, "rows")
    # (gradients in the logits' 16-bit type: a rounding each side of another sum)
    _close(sum(s[2].float() for _, s in got), dh, 2.0 ** -6 * float(dh.abs().max()), 0.0, "dh")
    _close(torch.cat([s[3] for _, s in got]), dw, 2.0 ** -6 * float(dw.abs().max()), 0.0, "dW")


def test_a_shard_needs_its_group():
    ops = _ops()
    x, tokens = torch.randn(3, 64, device=DEV).bfloat16(), torch.tensor([71, 72, 73], device=DEV)
    ids, logq = _teacher(3, 64, 2)
    h, W = torch.randn(3, 64, device=DEV).bfloat16(), torch.randn(64, 64, device=DEV).bfloat16()
    for call in (lambda: ops.token_logprobs(x, tokens, vocab_start=64),
                 lambda: ops.topk_distill_loss(x, ids, logq, denom=3.0, vocab_start=64),
                 lambda: ops.fused_lm_head_token_logprobs(h, W, tokens, vocab_start=64),
                 lambda: ops.fused_lm_head_topk_distill(h, W, ids, logq, denom=3.0, vocab_start=64)):
        with pytest.raises(ValueError, match="vocab_start"):
            call()


# ------------------------------------------------------------------------------------- every column's gradient
def _check_columns(got, want, bound, dtype):
    """`bound` of every element, before the rounding to the type."""
    limit = bound + 1.01 * ROUND[dtype] * want.abs() + TINY[dtype]
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), (float((off / limit).max()), torch.nonzero(off > limit)[0].tolist())
    assert float(((got == 0) & (want.abs() > 4 * TINY[dtype])).double().mean()) == 0.0


def _long_rows(rows, vocab, dtype, kind, view):
    x = _logits(rows, vocab + 9, dtype, seed=vocab + rows, spread=3.0 if kind == "spread" else 0.05)
    if kind == "flat":
        x = (x.float() * 0.1).to(dtype)
    return x[:, 9:] if view == "offset" else x[:, :vocab].contiguous()


COLUMNS = [(3, 151936), (40, 60013), (260, 50021), (700, 20011), (5, 1003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,view", [("flat", "whole"), ("spread", "whole"), ("flat", "offset")])
@pytest.mark.parametrize("rows,vocab", COLUMNS)
def test_every_column_of_the_scores_gradient(rows, vocab, dtype, kind, view):
    """An element is p times factors: t = x c - R to 2 x 2^-24 |t|, |t| <= 60, makes e right to 5e-6; the exponential, 1 / s
    and four products add 3e-6.  The entropy's factor ln p + H is right to that of its two terms and 4e-5."""
    x = _long_rows(rows, vocab, dtype, kind, view).requires_grad_()
    g = torch.Generator(device=DEV).manual_seed(4)
    tokens = torch.randint(0, vocab, (rows, 2), device=DEV, generator=g)
    up = 4096.0 if dtype == torch.float16 else 1.0
    d, dh = (up * torch.randn(rows, 2, device=DEV, generator=g), up * torch.randn(rows, device=DEV, generator=g))
    r = _ops().token_logprobs(x, tokens, 0.9)
    (got,) = torch.autograd.grad((r.logp, r.entropy), x, (d, dh))
    want = oracle.token_grad(x.detach(), tokens, 0.9, d, dh)
    logp = oracle.log_softmax(oracle.scaled(x.detach(), 0.9))
    p, D, H = logp.exp(), d.double().abs(), dh.double().abs()[:, None]
    terms = 8e-6 * (D.sum(1, keepdim=True) + H * (logp.abs() - (p * logp).sum(1, keepdim=True))) + 4e-5 * H
    bound = (p * terms).scatter_add_(1, tokens, D * 2.0 ** -22) / 0.9
    _check_columns(got, want, bound, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,view", [("flat", "whole"), ("spread", "whole"), ("flat", "offset")])
@pytest.mark.parametrize("rows,vocab", COLUMNS)
@pytest.mark.parametrize("tail", [True, False])
def test_every_column_of_the_distillation_gradient(rows, vocab, dtype, kind, view, tail):
    """Outside the entries (Q - q_r / p_r) p, its parts as right as those of the scores' gradient; on them Q p - q."""
    x = _long_rows(rows, vocab, dtype, kind, view).requires_grad_()
    ids, logq = _teacher(rows, vocab, 24)
    up = 4096.0 if dtype == torch.float16 else 1.0
    loss, _ = _ops().topk_distill_loss(x, ids, logq, denom=1.0, temperature=0.9, tail=tail, grad_scale=up)
    (got,) = torch.autograd.grad(loss, x, torch.tensor(up, device=DEV))
    _, want = oracle.distill(x.detach(), ids, logq, 0.9, tail)
    p = oracle.log_softmax(oracle.scaled(x.detach(), 0.9)).exp()
    q = torch.zeros_like(p).scatter_(1, ids, logq.double().exp())
    if tail:
        rest = p.scatter(1, ids, 0.0).sum(1, keepdim=True)
        factor = 1.0 + (1.0 - q.sum(1, keepdim=True)) / rest
    else:
        q, factor = q / q.sum(1, keepdim=True), 1.0
    _check_columns(got, want * up, 8e-6 * up * (p * factor + q) / 0.9, dtype)
    if view == "whole" and dtype != torch.float16:
        from bridge_b200.ops._ext import kernels

        own = x.detach().clone()
        kernels().distill_rows_inplace(own, ids, logq, None, None, 0.9, 1.0, tail, True)
        assert torch.equal(own, got)


@pytest.mark.parametrize("main", [True, False])
@pytest.mark.parametrize("rows", [1, 200, 256, 257, 700])
def test_head_gradients_kept_either_way(main, rows):
    """Up to 2 H = 256 rows of BF16 keep the chunks' gradients for the backward, more of them the weight's."""
    h, W, ids, logq, w = _head(U=rows)
    h.requires_grad_()
    W.requires_grad_()
    if main:
        W.main_grad = torch.full(W.shape, 2.0, device=DEV)
    loss, _ = _ops().fused_lm_head_topk_distill(h, W, ids, logq, denom=float(rows), weights=w, chunk_rows=96)
    assert not main or bool((W.main_grad == 2.0).all())
    (loss * 0.3).backward(retain_graph=True)
    loss.backward()
    hd, Wd = h.detach().double(), W.detach().double()
    _, gx = oracle.distill(hd @ Wd.t(), ids, logq, 1.0, True)
    gx = gx * w.double()[:, None] * 1.3 / rows
    dh, dw = gx @ Wd, gx.t() @ hd
    got = W.main_grad - 2.0 if main else W.grad
    _close(h.grad, dh, 2e-2 * float(dh.abs().max()), 5e-2, "dh")
    _close(got, dw, 2e-2 * float(dw.abs().max()), 5e-2, "dW")


@pytest.mark.parametrize("vocab", [300, 70001])
@pytest.mark.parametrize("fill", [-1e10, -1e20])
def test_tokens_under_a_finite_mask_keep_their_log_probs(vocab, fill):
    """In a row with live logits a filled token has the log-prob of its fill, and a teacher's entry there costs as much."""
    x = _logits(4, vocab, torch.float32)
    x[:, 7:60] = fill
    tokens = torch.tensor([[7, 3], [8, 9], [59, 60], [30, 0]], device=DEV)
    r = _ops().token_logprobs(x, tokens, 0.8)
    _check_logp(r, x, tokens, 0.8)
    assert bool(torch.isfinite(r.logp).all())
    y = torch.full((4, vocab), fill, device=DEV)
    y[:, 5] = 1.0
    r = _ops().token_logprobs(y, None, 0.8, top_k=3)
    _check_top(r, y, 0.8, 3)
    assert bool(torch.isfinite(r.top_logp).all())
    logq = torch.full((4, 2), -1.0, device=DEV)
    for tail in (True, False):
        _check_distill(x, tokens, logq, tail=tail, temp=0.8)


def test_tokens_under_a_finite_mask_in_shards(monkeypatch):
    x = _logits(4, 900, torch.float32)
    x[:, 250:800] = -1e10
    tokens = torch.tensor([[7, 300], [8, 799], [59, 250], [899, 0]], device=DEV)
    logq = torch.full((4, 2), -1.0, device=DEV)

    def work(rank, group):
        mine = x[:, rank * 300:(rank + 1) * 300].contiguous()
        at = dict(vocab_start=rank * 300, tp_group=group)
        return (_ops().token_logprobs(mine, tokens, 0.8, **at),
                _ops().topk_distill_loss(mine, tokens, logq, denom=1.0, temperature=0.8, **at)[1])

    kl, _ = oracle.distill(x, tokens, logq, 0.8, True)
    for r, rows in _ranks(monkeypatch, 3, work):
        _check_logp(r, x, tokens, 0.8)
        _close(rows, kl, 1e-5, 2e-6, "rows")
