"""The PyTorch form of the operators over rows of logits where it can go wrong."""

import math

import pytest
import torch

from bridge_b200.ops import (fused_lm_head_token_logprobs, fused_lm_head_topk_distill, token_logprobs,
                             topk_distill_loss)
from tests import vocab_oracle as oracle
from tests.dist_utils import run_ranks


def test_rows_of_finite_masks_carry_nothing():
    for fill in (-1e10, -1e15, -1e25):
        x = torch.full((2, 30), fill).requires_grad_()
        r = token_logprobs(x, torch.tensor([1, 2]), top_k=3)
        assert r.logp.tolist() == [-math.inf] * 2 and r.entropy.tolist() == [0.0] * 2
        (g,) = torch.autograd.grad((r.logp, r.entropy), x, (torch.ones(2), torch.ones(2)))
        assert not g.any()
    x = torch.zeros(2, 30)
    x[1, 4] = 3e10
    assert torch.isnan(token_logprobs(x, torch.tensor([1, 4])).logp).tolist() == [False, True]


# ------------------------------------------------------------------------------------------------ heads
def _stand_in(monkeypatch):
    """The head-level autograd nodes on the CPU: the kernels' calls in the PyTorch form."""
    from bridge_b200.ops import distill

    class Kernels:
        @staticmethod
        def distill_rows_inplace(lg, ids, logq, weights, temp, temp1, scale, tail, want):
            stats, xc = distill._open_reference(lg, ids, temp, temp1, 0)
            rows, coef, fix = distill._finish_reference(stats, xc, ids, logq, weights, temp, temp1, scale, tail,
                                                        lg.shape[1])
            if want:
                lg.copy_(distill._grad_reference(lg, ids, coef, fix, temp, temp1, 0, lg.shape[1]))
            return rows.float()

        @staticmethod
        def distill_open(logits, ids, logq, weights, temp, temp1, start, total):
            return distill._open_reference(logits, ids, temp, temp1, start)

        distill_finish = staticmethod(distill._finish_reference)

        @staticmethod
        def distill_grad(logits, ids, coef, fix, temp, temp1, start, total, inplace):
            return distill._grad_reference(logits, ids, coef, fix, temp, temp1, start, total)

        @staticmethod
        def weighted_rows_sum(rows, weights, denom):
            return (rows if weights is None else rows * weights).sum() / denom

    monkeypatch.setattr(distill, "on_gpu", lambda *t: True)
    monkeypatch.setattr(distill, "kernels", lambda: Kernels)


def _head(U=40, H=16, V=60, K=5, dtype=torch.float32):
    g = torch.Generator().manual_seed(3)
    h = torch.randn(U, H, generator=g).to(dtype).requires_grad_()
    W = torch.randn(V, H, generator=g).to(dtype).requires_grad_()
    top = torch.topk(torch.log_softmax(2 * torch.randn(U, V, generator=g), 1), K, dim=1)
    return h, W, top.indices, top.values


def test_head_loss_without_gradient_leaves_main_grad_alone(monkeypatch):
    _stand_in(monkeypatch)
    h, W, ids, logq = _head()
    W.main_grad = torch.zeros(W.shape)
    with torch.no_grad():
        loss, rows = fused_lm_head_topk_distill(h, W, ids, logq, denom=40.0, chunk_rows=16)
    assert not W.main_grad.any()
    assert torch.allclose(rows.double(), oracle.distill((h @ W.t()).detach(), ids, logq, 1.0, True)[0], atol=1e-4)


def _head_gradients(h, W, ids, logq, factor):
    """In 64 bits, of ``factor`` times the loss."""
    x = (h.detach().double() @ W.detach().double().t())
    _, gx = oracle.distill(x, ids, logq, 1.0, True)
    gx = gx * factor / h.shape[0]
    return gx @ W.detach().double(), gx.t() @ h.detach().double()


@pytest.mark.parametrize("main", [True, False])
@pytest.mark.parametrize("announced,factor", [(1.0, 1.0), (1.0, 0.5), (4.0, 4.0), (4.0, 3.0)])
def test_head_gradients_agree_for_any_loss_factor(monkeypatch, main, announced, factor):
    _stand_in(monkeypatch)
    h, W, ids, logq = _head()
    if main:
        W.main_grad = torch.full(W.shape, 2.0)
    loss, _ = fused_lm_head_topk_distill(h, W, ids, logq, denom=40.0, chunk_rows=16, grad_scale=announced)
    assert not main or bool((W.main_grad == 2.0).all())         # nothing happens to it before the backward
    (loss * factor).backward(retain_graph=True)
    dh, dw = _head_gradients(h, W, ids, logq, factor)
    got = W.main_grad - 2.0 if main else W.grad
    assert torch.allclose(h.grad.double(), dh, atol=1e-5, rtol=1e-4)
    assert torch.allclose(got.double(), dw, atol=1e-5, rtol=1e-4)
    loss.backward()                                              # and once more: gradients add up
    both = _head_gradients(h, W, ids, logq, factor + 1.0)
    got = W.main_grad - 2.0 if main else W.grad
    assert torch.allclose(h.grad.double(), both[0], atol=1e-5, rtol=1e-4)
    assert torch.allclose(got.double(), both[1], atol=1e-5, rtol=1e-4)


@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_head_counts_once(monkeypatch, reentrant):
    from torch.utils.checkpoint import checkpoint

    _stand_in(monkeypatch)
    h, W, ids, logq = _head()
    W.main_grad = torch.zeros(W.shape)
    loss = checkpoint(lambda v: fused_lm_head_topk_distill(v, W, ids, logq, denom=40.0, chunk_rows=16)[0], h,
                      use_reentrant=reentrant)
    loss.backward()
    dh, dw = _head_gradients(h, W, ids, logq, 1.0)
    assert torch.allclose(h.grad.double(), dh, atol=1e-5) and torch.allclose(W.main_grad.double(), dw, atol=1e-5)


# ---------------------------------------------------------------------------------------- loss factors
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_unannounced_loss_scale_is_applied_before_rounding(dtype):
    """A gradient that underflows unscaled, as a loss scaler meets it: one rounding, of the scaled gradient."""
    g = torch.Generator().manual_seed(0)
    x = (3.0 * torch.randn(16, 1024, generator=g)).to(dtype).requires_grad_()
    top = torch.topk(torch.log_softmax(2 * torch.randn(16, 1024, generator=g), 1), 8, dim=1)
    for scale in (16384.0, 98304.0):
        loss, _ = topk_distill_loss(x, top.indices, top.values, denom=4096.0)
        (got,) = torch.autograd.grad(loss * scale, x)
        _, want = oracle.distill(x.detach(), top.indices, top.values, 1.0, True)
        want = want * scale / 4096.0
        # the type's rounding, and 4e-6 (FP32 arithmetic) of the terms that cancel: p, and q on the given tokens
        q = torch.zeros_like(want).scatter_(1, top.indices, top.values.double().exp())
        terms = (torch.softmax(x.detach().double(), 1) + q) * scale / 4096.0
        rounding = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
        bound = 1.01 * rounding * want.abs() + 4e-6 * terms + 2.0 ** -25
        assert bool(((got.double() - want).abs() <= bound).all())
        if dtype == torch.float16:
            assert int((got == 0).sum()) < 0.05 * got.numel()


@pytest.mark.parametrize("main", [True, False])
def test_head_unannounced_loss_scale_in_fp16(monkeypatch, main):
    """Gradients of FP16 logits under a head, which underflow unscaled: FP16 matrix products of what is rounded once."""
    _stand_in(monkeypatch)
    h, W, ids, logq = _head(dtype=torch.float16)
    h, W = (0.25 * h).detach().requires_grad_(), (0.25 * W).detach().requires_grad_()
    if main:
        W.main_grad = torch.zeros(W.shape)
    scale = 2.0 ** 20
    loss, _ = fused_lm_head_topk_distill(h, W, ids, logq, denom=2.0 ** 25, chunk_rows=16)
    (loss * scale).backward()
    dh, dw = _head_gradients(h, W, ids, logq, scale * 40.0 / 2.0 ** 25)
    # 60 and 40 products of at most 1/32 x 1, each with a rounding of the logits (2^-11 of 4) and its own: below 2^-6 of the
    # largest, where the underflow of what is below 2^-25 took everything
    assert float((h.grad.double() - dh).abs().max()) <= 2.0 ** -6 * float(dh.abs().max())
    got = W.main_grad if main else W.grad
    assert float((got.double() - dw).abs().max()) <= 2.0 ** -6 * float(dw.abs().max())


# -------------------------------------------------------------------------------- no second derivative
def test_second_derivatives_are_refused(monkeypatch):
    x = torch.randn(3, 20, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([1, 2, 3])
    ids, logq = torch.tensor([[0, 4]] * 3), torch.full((3, 2), -1.5)
    r = token_logprobs(x, tokens)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x, create_graph=True)
    loss, _ = topk_distill_loss(x, ids, logq, denom=3.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, x, create_graph=True)
    _stand_in(monkeypatch)
    h, W, ids, logq = _head()
    loss, _ = fused_lm_head_topk_distill(h, W, ids, logq, denom=40.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, h, create_graph=True)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(3, 20), torch.randn(3, 20))
        with pytest.raises((RuntimeError, NotImplementedError)):
            token_logprobs(x, torch.tensor([1, 2, 3]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            topk_distill_loss(x, torch.tensor([[0, 4]] * 3), torch.full((3, 2), -1.5), denom=3.0)


# --------------------------------------------------------------------------- teachers that cover all that lives
def _covered(rows=16, vocab=120, live=40, device="cpu", seed=0):
    """Teacher and student under the same mask, which leaves fewer tokens than the teacher gives alternatives."""
    g = torch.Generator().manual_seed(seed)
    t, x = (3.0 * torch.randn(rows, vocab, generator=g) for _ in range(2))
    for u in range(rows):
        gone = torch.randperm(vocab, generator=g)[live:]
        t[u, gone] = x[u, gone] = -math.inf
    return t.to(device), x.to(device)


def _kl_of_live(t, x, temp=1.0):
    lq, lp = torch.log_softmax(t.double() / temp, 1), torch.log_softmax(x.double() / temp, 1)
    q, p = lq.exp(), lp.exp()
    return torch.where(q > 0, q * (lq - lp), torch.zeros_like(q)).sum(1), (p - q) / temp


def test_teacher_of_all_live_tokens_is_finite():
    """What FP32 log-probs leave of 1 is no probability where the student has none either: the KL of the live tokens."""
    t, x = _covered()
    teacher = token_logprobs(t, top_k=64)
    x.requires_grad_()
    loss, rows = topk_distill_loss(x, teacher.top_ids, teacher.top_logp, denom=16.0)
    want, grad = _kl_of_live(t, x.detach())
    assert torch.allclose(rows.double(), want, atol=1e-5) and bool(torch.isfinite(loss))
    assert torch.allclose(torch.autograd.grad(loss, x)[0].double(), grad / 16.0, atol=1e-6)
    # while mass that is really missing has nowhere to go
    _, rows = topk_distill_loss(x.detach(), teacher.top_ids, teacher.top_logp - 1e-3, denom=16.0)
    assert bool((rows == math.inf).all())


# ------------------------------------------------------------------------------------------- precision
def test_log_probs_keep_their_digits_far_from_zero():
    """FP32 logits around 60: a log-prob is right to 2e-6 and 2^-21 of its size, not to the logits' last place."""
    g = torch.Generator().manual_seed(2)
    x = 60.0 + torch.randn(50, 300, generator=g)
    tokens = torch.randint(0, 300, (50, 2), generator=g)
    r = token_logprobs(x, tokens, 0.7, top_k=5)
    want, ent = oracle.token_logprobs(x, tokens, 0.7)
    assert r.logp.dtype == r.entropy.dtype == r.top_logp.dtype == torch.float32
    assert bool(((r.logp.double() - want).abs() <= 2e-6 + 5e-7 * want.abs()).all())
    top, _ = oracle.token_logprobs(x, r.top_ids, 0.7)
    assert bool(((r.top_logp.double() - top).abs() <= 2e-6 + 5e-7 * top.abs()).all())
    assert bool(((r.entropy.double() - ent).abs() <= 4e-5).all())


# -------------------------------------------------------------------------------------------- refusals
def test_scoring_hidden_rows_checks_its_rows():
    """One token and one temperature a row; more of them were cut off in silence."""
    h, W = torch.randn(5, 16), torch.randn(30, 16)
    for bad in (dict(tokens=torch.zeros(6, dtype=torch.long)), dict(tokens=torch.zeros(4, dtype=torch.long)),
                dict(temperature=torch.ones(6)), dict(temperature=torch.ones(5, 1)),
                dict(tokens=torch.zeros(5, 2, 2, dtype=torch.long))):
        for chunk in (2, 3, 4096):
            with pytest.raises(ValueError):
                fused_lm_head_token_logprobs(h, W, chunk_rows=chunk, **bad)
    with pytest.raises(TypeError):
        fused_lm_head_token_logprobs(h, W, torch.zeros(5))
    r = fused_lm_head_token_logprobs(h, W, torch.zeros(5, dtype=torch.long), torch.ones(5), chunk_rows=2)
    assert r.logp.shape == (5,)


def test_a_shard_needs_its_group():
    """A first token other than 0 says that the logits are a shard, whose rows mean nothing alone."""
    x, tokens, ids = torch.randn(3, 20), torch.tensor([21, 22, 23]), torch.tensor([[21, 24]] * 3)
    logq, h, W = torch.full((3, 2), -1.5), torch.randn(3, 16), torch.randn(20, 16)
    for call in (lambda: token_logprobs(x, tokens, vocab_start=20),
                 lambda: topk_distill_loss(x, ids, logq, denom=3.0, vocab_start=20),
                 lambda: fused_lm_head_token_logprobs(h, W, tokens, vocab_start=20),
                 lambda: fused_lm_head_topk_distill(h, W, ids, logq, denom=3.0, vocab_start=20)):
        with pytest.raises(ValueError, match="vocab_start"):
            call()


# ------------------------------------------------------------------------------- tensor-parallel models
def _model_worker(rank, world):
    import torch.distributed as dist

    from bridge_b200.models import build_model, get_config
    from bridge_b200.rl import distill_loss, teacher_alternatives

    cfg = get_config("tiny")
    teacher, student = (build_model(cfg, seed=s, tp_group=dist.group.WORLD, dtype=torch.float32) for s in (1, 2))
    g = torch.Generator().manual_seed(0)
    h = torch.randn(9, cfg.hidden_size, generator=g).requires_grad_()
    ids, logp = teacher_alternatives(teacher, h.detach(), top_k=12, temperature=0.8)
    loss, rows = distill_loss(student, h, ids, logp, denom=9.0, temperature=0.8)
    (3.0 * loss).backward()
    return [v.detach().tolist() for v in (teacher.head_weight, student.head_weight, h, ids, logp, loss, rows, h.grad,
                                          student.head_weight.grad)]


def test_distillation_of_tensor_parallel_models():
    """Every rank of two vocabulary-parallel models gets the whole alternatives, loss and ``dh``, and its head's part."""
    ranks = [[torch.tensor(v) for v in r] for r in run_ranks(2, _model_worker)]
    wt, ws = (torch.cat([r[i] for r in ranks]).double() for i in (0, 1))
    h = ranks[0][2].double()
    ids = oracle.top(h @ wt.t(), 12)
    logq = oracle.token_logprobs(h @ wt.t(), ids, 0.8)[0]
    kl, gx = oracle.distill(h @ ws.t(), ids, logq, 0.8, True)
    gx = gx * 3.0 / 9.0
    for r in ranks:
        assert torch.equal(r[3], ids) and torch.allclose(r[4].double(), logq, atol=1e-5)
        assert torch.allclose(r[5].double(), kl.mean(), atol=1e-5) and torch.allclose(r[6].double(), kl, atol=1e-5)
        assert torch.allclose(r[7].double(), gx @ ws, atol=1e-5)
    assert torch.allclose(torch.cat([r[8] for r in ranks]).double(), gx.t() @ h, atol=1e-5)


@pytest.mark.parametrize("main", [True, False])
@pytest.mark.parametrize("rows", [1, 16, 17, 40])
@pytest.mark.parametrize("chunk", [7, 64])
def test_head_gradients_kept_either_way(monkeypatch, main, rows, chunk):
    """Few rows keep the chunks' gradients for the backward (up to 16 of FP32 here), many the weight's."""
    _stand_in(monkeypatch)
    h, W, ids, logq = _head(U=rows)
    if main:
        W.main_grad = torch.full(W.shape, 2.0)
    loss, _ = fused_lm_head_topk_distill(h, W, ids, logq, denom=float(rows), chunk_rows=chunk)
    assert not main or bool((W.main_grad == 2.0).all())
    (loss * 0.3).backward()
    dh, dw = _head_gradients(h, W, ids, logq, 0.3)
    got = W.main_grad - 2.0 if main else W.grad
    assert torch.allclose(h.grad.double(), dh, atol=1e-5, rtol=1e-4)
    assert torch.allclose(got.double(), dw, atol=1e-5, rtol=1e-4)


def test_tokens_under_a_finite_mask_keep_their_log_probs():
    x = torch.randn(4, 60)
    x[:, 7:40] = -1e10
    tokens = torch.tensor([[7, 3], [8, 9], [39, 40], [30, 0]])
    r = token_logprobs(x, tokens, 0.8)
    want, _ = oracle.token_logprobs(x, tokens, 0.8)
    assert bool(((r.logp.double() - want).abs() <= 2e-6 + 5e-7 * want.abs()).all())
    logq = torch.full((4, 2), -1.0)
    for tail in (True, False):
        _, rows = topk_distill_loss(x, tokens, logq, denom=1.0, tail=tail)
        kl, _ = oracle.distill(x, tokens, logq, 1.0, tail)
        assert bool(((rows.double() - kl).abs() <= 1e-5 + 2e-6 * kl.abs()).all())
    _, rows = topk_distill_loss(torch.full((4, 60), -1e10), tokens, logq, denom=1.0)
    assert rows.tolist() == [math.inf] * 4
