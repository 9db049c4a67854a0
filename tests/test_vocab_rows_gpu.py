"""Kernels over rows of logits against their 64-bit definitions: token log-probs with entropy and alternatives,
and distillation from a teacher's top log-probs, forward and backward.

Tolerances.  A term 2^t carries the error of t (2^-24 |t|, |t| < 32 wherever a term counts) and of the exponential
(2^-22): under 2e-6, and log s with it; a log-prob adds its own rounding and that of log2(e)/T, 2^-23 of its size.
The entropy is a mean of t over such terms: 32 times as much in the worst case, 4e-5.  A gradient is p times factors
of that accuracy, rounded once to the output's type.
"""

import math

import pytest
import torch

from tests import vocab_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}


def _ops():
    from bridge_b200 import ops

    return ops


def _logits(rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab, device=DEV, generator=g) * spread
    if vocab > 4 and rows:
        x[:, :: max(1, vocab // 5)] += 6.0
    return x.to(dtype)


def _close(got, want, atol, rtol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~(off <= atol + rtol * want.abs())
    assert not bool(bad.any()), f"{what}: {float(off[bad].max()) if bad.any() else 0} at {torch.nonzero(bad)[0].tolist()}"


def _check_logp(r, x, tokens, temp):
    want, ent = oracle.token_logprobs(x, tokens, temp)
    if tokens is not None:
        _close(r.logp.view(want.shape), want, 2e-6, 5e-7, "logp")
    if r.entropy is not None:
        _close(r.entropy, ent, 4e-5, 5e-7, "entropy")


def _check_top(r, x, temp, k):
    ids = oracle.top(x, k)
    assert torch.equal(r.top_ids, ids)
    want, _ = oracle.token_logprobs(x, ids, temp)
    _close(r.top_logp, want, 2e-6, 5e-7, "top_logp")


def _check_grad(got, want, size, dtype):
    """`size` [U, 1] bounds the terms that cancel in a row's gradient (times T)."""
    assert got.dtype == dtype
    bound = 4e-6 * size + ROUND[dtype] * want.abs() * 1.01 + TINY[dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# --------------------------------------------------------------------------------------- token log-probs
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 8, 8), (4, 9, 1), (3, 127, 20),
                                          (2, 1000, 256), (7, 4099, 64), (3, 32003, 128), (2, 151936, 20),
                                          (70, 5003, 5), (300, 1024, 8)])
def test_token_logprobs(dtype, rows, vocab, k):
    x = _logits(rows, vocab, dtype, seed=vocab)
    g = torch.Generator(device=DEV).manual_seed(1)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    temp = 0.5 + torch.rand(rows, device=DEV, generator=g)
    r = _ops().token_logprobs(x, tokens, temp, top_k=k)
    _check_logp(r, x, tokens[:, None], temp)
    _check_top(r, x, temp, k)
    only = _ops().token_logprobs(x, None, temp, top_k=k, with_entropy=False)
    assert only.logp is None and only.entropy is None
    assert torch.equal(only.top_ids, r.top_ids) and torch.equal(only.top_logp, r.top_logp)
    assert _ops().token_logprobs(x, tokens, 1.0).top_ids is None


@pytest.mark.parametrize("rows", [1, 5, 37, 148, 149, 600, 2500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_row_counts(rows, dtype):
    """Every way of splitting rows over blocks."""
    x = _logits(rows, 9001, dtype, seed=rows)
    tokens = torch.randint(0, 9001, (rows, 3), device=DEV)
    r = _ops().token_logprobs(x, tokens, 0.9, top_k=33)
    _check_logp(r, x, tokens, 0.9)
    _check_top(r, x, 0.9, 33)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("view", ["offset", "odd_stride", "columns", "expanded"])
def test_token_logprobs_strides(dtype, view):
    rows, vocab = 6, 3001
    if view == "offset":
        x = _logits(rows, vocab + 16, dtype)[:, 3:3 + vocab]
    elif view == "odd_stride":
        x = _logits(rows, vocab + 2, dtype)[:, :vocab]
    elif view == "columns":
        x = _logits(vocab, rows, dtype).t()
    else:
        x = _logits(1, vocab, dtype).expand(rows, vocab)
    x = x.detach().requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device=DEV)
    r = _ops().token_logprobs(x, tokens, top_k=9)
    _check_logp(r, x.detach(), tokens[:, None], 1.0)
    _check_top(r, x.detach(), 1.0, 9)
    d = torch.randn(rows, device=DEV)
    (got,) = torch.autograd.grad(r.logp, x, d)
    want = oracle.token_grad(x.detach(), tokens[:, None], 1.0, d[:, None], None)
    _check_grad(got, want, d.abs()[:, None].double(), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("units", [1, 31, 128, 129, 1023, 1024, 1025, 2047, 2048, 4100, 8191, 16384, 16400])
def test_scores_alone_at_batch_edges(dtype, units):
    """Lengths around a warp's, a block's and a cluster's batches; rows at every offset from 16 bytes, with masked ends."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    for rows, short, offset in ((3, 0, 0), (9, 1, 1), (40, per - 1, per - 1)):
        vocab = max(1, units * per - short)
        x = _logits(rows, vocab + per + 1, dtype, seed=units)[:, offset:offset + vocab]
        x[0, vocab // 2:] = -math.inf
        x[1, : vocab // 2] = torch.finfo(dtype).min
        tokens = torch.randint(0, vocab, (rows,), device=DEV)
        tokens[0] = 0 if vocab > 1 else -1
        tokens[1] = vocab - 1
        tokens[2] = vocab - 1
        r = _ops().token_logprobs(x, tokens, 1.3)
        _check_logp(r, x, tokens[:, None], 1.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 12, 70, 101])
def test_long_rows_held_or_streamed(dtype, rows):
    """Few long rows: alternatives and distillation in registers or streamed, as row count and type decide."""
    vocab = 100003
    x = _logits(rows, vocab, dtype, seed=rows)
    tokens = torch.randint(0, vocab, (rows,), device=DEV)
    r = _ops().token_logprobs(x, tokens, 1.1, top_k=17)
    _check_logp(r, x, tokens[:, None], 1.1)
    _check_top(r, x, 1.1, 17)
    ids, logq = _teacher(rows, vocab, 17)
    _check_distill(x, ids, logq, tail=True, denom=float(rows))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(dtype):
    """Masks of -inf and of the type's lowest value, a row with one live logit, rows with none."""
    vocab = 777
    x = _logits(6, vocab, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0, 100:] = -math.inf
    x[1, :700] = low
    x[2] = -math.inf
    x[2, 500] = 1.5
    x[3] = -math.inf
    x[4] = low
    x[5, ::2] = -math.inf
    x[5, 1::4] = low
    x = x.requires_grad_()
    tokens = torch.tensor([[5, 300], [750, 3], [500, 0], [1, 2], [1, 2], [3, 2]], device=DEV)
    r = _ops().token_logprobs(x, tokens, top_k=12)
    _check_logp(r, x.detach(), tokens, 1.0)
    _check_top(r, x.detach(), 1.0, 12)
    d, dh = torch.randn(6, 2, device=DEV), torch.randn(6, device=DEV)
    (got,) = torch.autograd.grad((r.logp, r.entropy), x, (d, dh))
    want = oracle.token_grad(x.detach(), tokens, 1.0, d, dh)
    size = (d.abs().sum(1) + 32 * dh.abs())[:, None].double()
    _check_grad(got, want, size, dtype)
    # (the lowest FP16 value is a number like any other)
    for dead in ((3, 4) if dtype != torch.float16 else (3,)):
        assert bool((r.logp[dead] == -math.inf).all()) and float(r.entropy[dead].detach()) == 0.0
        assert bool((got[dead] == 0).all()) and r.top_ids[dead].tolist() == list(range(12))


def test_nan_and_infinite_logits():
    x = _logits(3, 500, torch.float32)
    x[0, 17] = math.nan
    x[1, 3] = math.inf
    r = _ops().token_logprobs(x, torch.tensor([1, 2, 3], device=DEV), top_k=4)
    assert bool(torch.isnan(r.logp[:2]).all()) and bool(torch.isnan(r.entropy[:2]).all())
    assert torch.equal(r.top_ids, oracle.top(x, 4))
    assert bool(torch.isfinite(r.logp[2]))
    x[:] = math.nan
    r = _ops().token_logprobs(x, None, top_k=256)
    assert torch.equal(r.top_ids, torch.arange(256, device=DEV).expand(3, 256))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [6000, 40001])
@pytest.mark.parametrize("kind", ["equal", "two_values", "few_live", "rising", "falling", "one_stripe", "signed_zero",
                                  "block", "quantised"])
def test_alternatives_in_hard_rows(dtype, vocab, kind):
    """Ties without end, sorted rows, all large logits in the columns that one thread reads, less than k live."""
    rows = 3
    g = torch.Generator(device=DEV).manual_seed(5)
    if kind == "equal":
        x = torch.full((rows, vocab), 0.25, device=DEV)
    elif kind == "two_values":
        x = torch.zeros(rows, vocab, device=DEV)
        x[:, 3000:3090] = 1.0
    elif kind == "few_live":
        x = torch.full((rows, vocab), -math.inf, device=DEV)
        x[:, torch.tensor([4, 2999, vocab - 1], device=DEV)] = torch.tensor([1.0, 2.0, 1.0], device=DEV)
    elif kind == "rising":
        x = torch.linspace(-50, 50, vocab, device=DEV).expand(rows, vocab)
    elif kind == "falling":
        x = torch.linspace(50, -50, vocab, device=DEV).expand(rows, vocab)
    elif kind == "one_stripe":
        x = torch.randn(rows, vocab, device=DEV, generator=g)
        for period in (2048, 4096, 8192, 32768):
            for j in range(8):
                x[:, 8 + j::period] += 30.0
    elif kind == "signed_zero":
        x = torch.zeros(rows, vocab, device=DEV)
        x[:, ::3] = -0.0
    elif kind == "block":
        x = torch.randn(rows, vocab, device=DEV, generator=g)
        x[:, 1000:4500] += 20.0
    else:
        x = torch.randint(-3, 4, (rows, vocab), device=DEV, generator=g).float()
    x = x.to(dtype).contiguous()
    for k in (1, 40, 256):
        r = _ops().token_logprobs(x, None, 1.1, top_k=k)
        _check_top(r, x, 1.1, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,n", [(4, 9, 1), (3, 1000, 7), (2, 32003, 16), (260, 513, 2), (2, 151936, 1)])
@pytest.mark.parametrize("entropy", [True, False])
def test_token_logprobs_backward(dtype, rows, vocab, n, entropy):
    """Repeated tokens add up; padded positions (negative or past the vocabulary) have log-prob 0 and no gradient."""
    x = _logits(rows, vocab, dtype, seed=n).requires_grad_()
    g = torch.Generator(device=DEV).manual_seed(2)
    tokens = torch.randint(0, vocab, (rows, n), device=DEV, generator=g)
    if n > 2:
        tokens[:, 1] = tokens[:, 0]
        tokens[0, 2], tokens[1, 2] = -100, vocab
    temp = 0.5 + torch.rand(rows, device=DEV, generator=g)
    r = _ops().token_logprobs(x, tokens.int() if n == 7 else tokens, temp, with_entropy=entropy)
    _check_logp(r, x.detach(), tokens, temp)
    d = torch.randn(rows, n, device=DEV, generator=g)
    dh = torch.randn(rows, device=DEV, generator=g)
    if entropy:
        (got,) = torch.autograd.grad((r.logp, r.entropy), x, (d, dh))
    else:
        (got,) = torch.autograd.grad(r.logp, x, d)
    want = oracle.token_grad(x.detach(), tokens, temp, d, dh if entropy else None)
    size = ((d.abs().sum(1) + 32 * dh.abs() * entropy) / temp)[:, None].double()
    _check_grad(got, want, size, dtype)


def test_entropy_gradient_alone_and_empty_batch():
    x = _logits(5, 301, torch.float32).requires_grad_()
    r = _ops().token_logprobs(x)
    dh = torch.randn(5, device=DEV)
    (got,) = torch.autograd.grad(r.entropy, x, dh)
    _check_grad(got, oracle.token_grad(x.detach(), None, 1.0, None, dh), 32 * dh.abs()[:, None].double(), x.dtype)
    e = torch.empty(0, 301, device=DEV, requires_grad=True)
    r = _ops().token_logprobs(e, torch.empty(0, dtype=torch.long, device=DEV), top_k=3)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 3)
    (g,) = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), e)
    assert g.shape == (0, 301)


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit functions."""
    x = _logits(4, 203, torch.float32).requires_grad_()
    tokens = torch.randint(0, 203, (4, 2), device=DEV)
    way = torch.randn(4, 203, device=DEV)
    r = _ops().token_logprobs(x, tokens, 0.8)
    (g,) = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x)
    h = 1e-4

    def f(v):
        lp, ent = oracle.token_logprobs(v, tokens, 0.8)
        return float(lp.sum() + ent.sum())

    xd = x.detach().double()
    num = (f(xd + h * way) - f(xd - h * way)) / (2 * h)
    assert abs(float((g * way).double().sum()) - num) <= 1e-4 * max(1.0, abs(num))
    ids = torch.stack([torch.randperm(203, device=DEV)[:9] for _ in range(4)])
    logq = torch.log_softmax(torch.randn(4, 9, device=DEV), 1) - 0.3
    for tail in (True, False):
        loss, _ = _ops().topk_distill_loss(x, ids, logq, denom=1.0, temperature=0.8, tail=tail)
        (g,) = torch.autograd.grad(loss, x)

        def kl(v):
            return float(oracle.distill(v, ids, logq, 0.8, tail)[0].sum())

        num = (kl(xd + h * way) - kl(xd - h * way)) / (2 * h)
        assert abs(float((g * way).double().sum()) - num) <= 1e-4 * max(1.0, abs(num))


def test_offsets_beyond_32_bits():
    """The last rows of logits with more than 2^31 elements (4.3 GB)."""
    rows, vocab = 17000, 131072
    x = torch.zeros(rows, vocab, device=DEV, dtype=torch.bfloat16)
    tail = _logits(3, vocab, torch.bfloat16)
    x[-3:] = tail
    x.requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device=DEV)
    r = _ops().token_logprobs(x, tokens, top_k=5)
    want, ent = oracle.token_logprobs(tail, tokens[-3:, None], 1.0)
    _close(r.logp[-3:, None], want, 2e-6, 5e-7, "logp")
    assert torch.equal(r.top_ids[-3:], oracle.top(tail, 5))
    _close(r.logp[:5], torch.full((5,), -math.log(vocab), device=DEV), 2e-6, 5e-7, "logp")
    (g,) = torch.autograd.grad(r.logp, x, torch.ones(rows, device=DEV))
    wg = oracle.token_grad(tail, tokens[-3:, None], 1.0, torch.ones(3, 1, device=DEV), None)
    _check_grad(g[-3:], wg, torch.ones(3, 1, device=DEV, dtype=torch.float64), torch.bfloat16)


# ------------------------------------------------------------------------------------------ distillation
def _teacher(rows, vocab, k, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = 2.0 * torch.randn(rows, vocab, device=DEV, generator=g)
    top = torch.topk(t, k, dim=1)
    return top.indices, top.values - torch.logsumexp(t, dim=1, keepdim=True)


def _check_distill(x, ids, logq, *, tail, temp=1.0, weights=None, denom=3.0, grad_scale=1.0, upstream=1.0):
    x = x.detach().requires_grad_()
    loss, rows = _ops().topk_distill_loss(x, ids, logq, denom=denom, weights=weights, temperature=temp, tail=tail,
                                          grad_scale=grad_scale)
    kl, g = oracle.distill(x.detach(), ids, logq, temp, tail)
    w = torch.ones(x.shape[0], device=DEV, dtype=torch.float64) if weights is None else weights.double()
    kl = torch.where(w == 0, torch.zeros_like(kl), kl)
    _close(rows, kl, 4e-6, 1e-6, "rows")
    want = torch.where(w == 0, torch.zeros_like(kl), kl * w).sum() / denom
    _close(loss, want, 4e-6 * float(w.abs().sum()) / denom, 1e-6, "loss")
    (got,) = torch.autograd.grad(loss * upstream if upstream != 1.0 else loss, x)
    f = w[:, None] * upstream / denom
    it = (1.0 / temp.double())[:, None] if torch.is_tensor(temp) else 1.0 / temp
    _check_grad(got, torch.where(f == 0, torch.zeros_like(g), g * f), 2 * f.abs() * it, x.dtype)
    with torch.no_grad():
        again, rows2 = _ops().topk_distill_loss(x, ids, logq, denom=denom, weights=weights, temperature=temp,
                                                tail=tail)
    assert torch.equal(rows2, rows) and torch.equal(again, loss)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("rows,vocab,k", [(1, 2, 1), (3, 9, 4), (2, 8, 8), (5, 1000, 20), (3, 4099, 128),
                                          (2, 32003, 256), (2, 151936, 64), (200, 517, 16)])
def test_distill(dtype, tail, rows, vocab, k):
    x = _logits(rows, vocab, dtype, seed=k)
    ids, logq = _teacher(rows, vocab, k)
    g = torch.Generator(device=DEV).manual_seed(9)
    temp = 0.7 + torch.rand(rows, device=DEV, generator=g)
    weights = torch.rand(rows, device=DEV, generator=g) + 0.1
    up = 512.0 if dtype == torch.float16 else 1.0
    _check_distill(x, ids, logq, tail=tail, temp=temp, weights=weights, grad_scale=up, upstream=up)


@pytest.mark.parametrize("rows", [1, 6, 37, 148, 300, 1500])
@pytest.mark.parametrize("tail", [True, False])
def test_distill_row_counts(rows, tail):
    x = _logits(rows, 2999, torch.bfloat16, seed=rows)
    ids, logq = _teacher(rows, 2999, 24)
    _check_distill(x, ids, logq, tail=tail, denom=float(rows))


@pytest.mark.parametrize("tail", [True, False])
def test_distill_entries(tail):
    """Dropped entries, rows without any, repeated ids, an entry of probability 0, ids past the vocabulary."""
    x = _logits(7, 600, torch.float32)
    ids, logq = _teacher(7, 600, 10)
    ids[0, 4:] = -1
    ids[1] = -1
    ids[2, 5], ids[2, 9] = ids[2, 1], ids[2, 1]
    logq[3, 2] = -math.inf
    ids[4, 3], ids[4, 4] = 600, 10 ** 9
    ids[5, 1:] = -1
    got = _check_distill(x, ids, logq, tail=tail, denom=7.0)
    assert bool((got[1] == 0).all())
    _check_distill(x.bfloat16(), ids, logq, tail=tail, denom=7.0)


def test_distill_all_columns_given_and_full_teacher():
    """No column outside the entries; a teacher whose entries sum to 1 or, by rounding, to more."""
    x = _logits(3, 24, torch.float32)
    ids = torch.stack([torch.randperm(24, device=DEV) for _ in range(3)])
    logq = torch.log_softmax(torch.randn(3, 24, device=DEV), 1)
    for tail in (True, False):
        _check_distill(x, ids, logq, tail=tail)
    ids2, logq2 = ids[:, :6].contiguous(), torch.log_softmax(torch.randn(3, 6, device=DEV), 1) + 2e-7
    _check_distill(x, ids2, logq2, tail=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [True, False])
def test_distill_masked_logits(dtype, tail):
    """Masked columns carry nothing; where nothing is left outside the entries, or anywhere, nothing is NaN."""
    x = _logits(4, 400, dtype)
    ids, logq = _teacher(4, 400, 12)
    x[0, 200:] = -math.inf
    x[0].scatter_(0, ids[0], 1.0)
    x[1, 1::2] = torch.finfo(dtype).min
    x[1].scatter_(0, ids[1], 0.5)
    x[2, :] = 2.0
    x[3, 100:300] = -math.inf
    x[3].scatter_(0, ids[3], torch.zeros(12, device=DEV, dtype=dtype))
    up = 512.0 if dtype == torch.float16 else 1.0
    _check_distill(x, ids, logq, tail=tail, grad_scale=up, upstream=up)


def test_distill_without_student_probability():
    x = torch.randn(3, 100, device=DEV)
    ids, logq = _teacher(3, 100, 5)
    x[0, ids[0, 2]] = -math.inf                     # a given token that the student rules out
    keep = x[1].clone()
    x[1] = -math.inf
    x[1, ids[1]] = keep[ids[1]]                     # nothing outside the entries, while the teacher has some there
    x[2] = -math.inf                                # nothing at all
    x.requires_grad_()
    for tail in (True, False):
        loss, rows = _ops().topk_distill_loss(x, ids, logq, denom=1.0, tail=tail)
        assert rows[0] == math.inf and rows[2] == math.inf
        assert (rows[1] == math.inf) == tail
        (g,) = torch.autograd.grad(loss, x)
        assert not bool(torch.isnan(g).any()) and bool((g[2] == 0).all())


def test_distill_weight_zero_rows_are_not_read():
    x = _logits(4, 333, torch.bfloat16)
    x[1] = math.nan
    ids, logq = _teacher(4, 333, 6)
    weights = torch.tensor([1.0, 0.0, 0.5, 0.0], device=DEV)
    x2 = x.clone()
    x2[1] = 0.0
    got = _check_distill(x2, ids, logq, tail=True, weights=weights)
    x.requires_grad_()
    loss, rows = _ops().topk_distill_loss(x, ids, logq, denom=3.0, weights=weights)
    (g,) = torch.autograd.grad(loss, x)
    assert rows[1] == 0 and torch.equal(g, got) and bool((g[1] == 0).all())


def test_distill_far_tail():
    """A tail of 1e-40 of the student's probability still has its logarithm and its gradient."""
    x = torch.randn(2, 500, device=DEV)
    ids, logq = _teacher(2, 500, 4)
    x.scatter_(1, ids, 95.0)
    _check_distill(x, ids, logq, tail=True, denom=1.0)


def test_distill_unannounced_scale_and_second_backward():
    x = _logits(5, 700, torch.float32).requires_grad_()
    ids, logq = _teacher(5, 700, 6)
    loss, _ = _ops().topk_distill_loss(x, ids, logq, denom=5.0)
    (a,) = torch.autograd.grad(loss * 3.0, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="already taken"):
        torch.autograd.grad(loss, x)
    loss, _ = _ops().topk_distill_loss(x, ids, logq, denom=5.0)
    (b,) = torch.autograd.grad(loss, x)
    _close(a, 3.0 * b, 1e-12, 3e-7, "scaled")


@pytest.mark.parametrize("view", ["offset", "odd_stride", "columns", "expanded"])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_strides(dtype, view):
    rows, vocab = 5, 2501
    if view == "offset":
        x = _logits(rows, vocab + 16, dtype)[:, 5:5 + vocab]
    elif view == "odd_stride":
        x = _logits(rows, vocab + 2, dtype)[:, :vocab]
    elif view == "columns":
        x = _logits(vocab, rows, dtype).t()
    else:
        x = _logits(1, vocab, dtype).expand(rows, vocab)
    ids, logq = _teacher(rows, vocab, 11)
    up = 512.0 if dtype == torch.float16 else 1.0
    _check_distill(x, ids, logq, tail=True, grad_scale=up, upstream=up)


# --------------------------------------------------------------------------- shards, heads, streams, refusals
def _join(parts):
    top = torch.stack([p[0] for p in parts]).amax(0)
    s = sum(torch.exp2(p[0] - top) * p[1] for p in parts)
    et = sum(torch.exp2(p[0] - top) * (p[2] + torch.where(p[1] == 0, torch.zeros_like(top), p[0] - top) * p[1])
             for p in parts)
    return top, s, et


@pytest.mark.parametrize("dtype", TYPES)
def test_vocabulary_in_shards(dtype):
    """The open forms of the kernels, on three shards whose sums are joined here, against whole rows."""
    from bridge_b200.ops._ext import kernels

    m = kernels()
    rows, part = 9, 1001
    vocab = 3 * part
    x = _logits(rows, vocab, dtype)
    x[4, part:2 * part] = -math.inf
    cuts = [x[:, i * part:(i + 1) * part] for i in range(3)]
    tokens = torch.randint(0, vocab, (rows, 2), device=DEV)
    tokens[0, 1] = -1
    outs = [m.token_logprob_open(c, tokens, None, 0.9, 7, True, i * part) for i, c in enumerate(cuts)]
    r, s, et = _join([o[1].unbind(1) for o in outs])
    xt = sum(o[0] for o in outs)
    logp = math.log(2.0) * (xt.double() - r.double()[:, None] - torch.log2(s.double())[:, None])
    want, ent = oracle.token_logprobs(x, tokens, 0.9)
    ok = tokens >= 0
    _close(logp[ok], want[ok], 6e-6, 1e-6, "logp")
    _close(math.log(2.0) * (torch.log2(s.double()) - et.double() / s.double()), ent, 4e-5, 1e-6, "entropy")
    ids, top = torch.cat([o[2] for o in outs], 1), torch.cat([o[3] for o in outs], 1)
    at = m.token_logprob_open(top, None, None, 1.0, 7, False, 0)[2]
    assert torch.equal(ids.gather(1, at), oracle.top(x, 7))
    d, dh = torch.randn(rows, 2, device=DEV), torch.randn(rows, device=DEV)
    stats = torch.stack((r, 1.0 / s, et / s), 1)
    got = torch.cat([m.token_logprob_bwd(c, tokens, None, 0.9, stats, d, dh, i * part, vocab)
                     for i, c in enumerate(cuts)], 1)
    _check_grad(got, oracle.token_grad(x, tokens, 0.9, d, dh),
                2 * (d.abs().sum(1) + 32 * dh.abs())[:, None].double(), dtype)
    ids, logq = _teacher(rows, vocab, 18)
    ids[1, 9:] = -1
    ids[2, 3] = ids[2, 8]
    ids[3] = -1
    w = torch.rand(rows, device=DEV)
    w[5] = 0.0
    for tail in (True, False):
        outs = [m.distill_open(c, ids, logq, w, None, 0.9, i * part, vocab) for i, c in enumerate(cuts)]
        r, s, _ = _join([(o[0][:, 0], o[0][:, 1], torch.zeros(rows, device=DEV)) for o in outs])
        kl, coef, fix = m.distill_finish(torch.stack((r, s), 1), sum(o[1] for o in outs), ids, logq, w, None, 0.9,
                                         2.0, tail, vocab)
        kl_want, g_want = oracle.distill(x, ids, logq, 0.9, tail)
        live = w != 0
        _close(kl, torch.where(live, kl_want, torch.zeros_like(kl_want)), 1e-5, 2e-6, "rows")
        got = torch.cat([m.distill_grad(c, ids, coef, fix, None, 0.9, i * part, vocab, False)
                         for i, c in enumerate(cuts)], 1)
        f = (2.0 * w.double())[:, None]
        _check_grad(got, g_want * f, 4 * f, dtype)


@pytest.mark.parametrize("main_grad", [False, True])
def test_fused_head_distill_and_teacher(main_grad):
    """Teacher alternatives through its head, student loss through its own, against FP32 heads (tolerances of
    BF16 logits: 2^-9 of their size, and of BF16 gradients)."""
    ops = _ops()
    U, H, V, K = 300, 256, 5000, 16
    h = (torch.randn(U, H, device=DEV) * 0.5).bfloat16()
    W = (torch.randn(V, H, device=DEV) * 0.05).bfloat16()
    r = ops.fused_lm_head_token_logprobs(h, W, torch.zeros(U, dtype=torch.long, device=DEV), 0.8, top_k=K,
                                         chunk_rows=128)
    lp, ent = oracle.token_logprobs(h.float() @ W.float().t(), r.top_ids, 0.8)
    _close(r.top_logp, lp, 5e-2, 1e-2, "teacher")
    _close(r.entropy, ent, 5e-2, 1e-2, "entropy")
    hs = (h.float() + 0.3 * torch.randn(U, H, device=DEV)).bfloat16().requires_grad_()
    Ws = (W.float() + 0.01 * torch.randn(V, H, device=DEV)).bfloat16().requires_grad_()
    if main_grad:
        Ws.main_grad = torch.zeros(V, H, device=DEV)
    w = torch.rand(U, device=DEV)
    loss, rows = ops.fused_lm_head_topk_distill(hs, Ws, r.top_ids, r.top_logp, denom=float(U), weights=w,
                                                temperature=0.8, chunk_rows=128, grad_scale=4.0)
    (loss * 4.0).backward()
    hr, Wr = hs.detach().float().requires_grad_(), Ws.detach().float().requires_grad_()
    x = hr @ Wr.t()
    kl, g = oracle.distill(x.detach(), r.top_ids, r.top_logp, 0.8, True)
    _close(rows, kl, 5e-2, 1e-2, "rows")
    _close(loss, (kl * w.double()).sum() / U, 5e-3, 1e-2, "loss")
    x.backward((g * w.double()[:, None] * 4.0 / U).float())
    _close(hs.grad, hr.grad, 2e-3, 5e-2, "dh")
    _close(Ws.main_grad if main_grad else Ws.grad, Wr.grad, 2e-3, 5e-2, "dW")


def test_other_stream_and_determinism():
    x = _logits(64, 9001, torch.bfloat16)
    ids, logq = _teacher(64, 9001, 30)
    ops = _ops()
    base = ops.token_logprobs(x, None, top_k=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.token_logprobs(x, None, top_k=50)
        xs = x.detach().requires_grad_()
        loss, rows = ops.topk_distill_loss(xs, ids, logq, denom=64.0)
        (g,) = torch.autograd.grad(loss, xs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(base.top_ids, again.top_ids) and torch.equal(base.entropy, again.entropy)
    assert torch.equal(base.top_logp, again.top_logp)
    xs = x.detach().requires_grad_()
    loss2, rows2 = ops.topk_distill_loss(xs, ids, logq, denom=64.0)
    (g2,) = torch.autograd.grad(loss2, xs)
    assert torch.equal(rows, rows2) and torch.equal(loss, loss2) and torch.equal(g, g2)


def test_outputs_stay_inside():
    """In-place gradients between guard rows, and at an odd vocabulary where rows start off any boundary."""
    from bridge_b200.ops._ext import kernels

    for vocab, dtype in ((1003, torch.bfloat16), (1003, torch.float32), (1024, torch.bfloat16)):
        big = _logits(9, vocab, dtype)
        keep = big.clone()
        ids, logq = _teacher(7, vocab, 13)
        kernels().distill_rows_inplace(big[1:8], ids, logq, None, None, 1.0, 1.0, True, True)
        grad = big[1:8]
        assert torch.equal(big[0], keep[0]) and torch.equal(big[8], keep[8])
        _, want = oracle.distill(keep[1:8], ids, logq, 1.0, True)
        _check_grad(grad, want, torch.full((7, 1), 2.0, device=DEV, dtype=torch.float64), dtype)


def test_refusals():
    ops = _ops()
    x = torch.randn(3, 50, device=DEV)
    tok = torch.zeros(3, dtype=torch.long, device=DEV)
    for bad, err in ((dict(temperature=0.0), ValueError), (dict(temperature=-1.0), ValueError),
                     (dict(temperature=math.nan), ValueError), (dict(temperature=torch.ones(2, device=DEV)), ValueError),
                     (dict(temperature=torch.ones(3)), ValueError), (dict(top_k=51), ValueError),
                     (dict(top_k=-1), ValueError), (dict(tokens=tok[:2]), ValueError),
                     (dict(tokens=tok.float()), TypeError), (dict(tokens=tok.cpu()), ValueError),
                     (dict(tokens=tok.view(1, 3)), ValueError)):
        with pytest.raises(err):
            ops.token_logprobs(x, **bad)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.randn(3, 1000, device=DEV), top_k=257)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double())
    with pytest.raises(ValueError):
        ops.token_logprobs(x[0])
    ids, logq = _teacher(3, 50, 4)
    good = dict(denom=3.0)
    for change, err in ((dict(denom=0.0), ValueError), (dict(grad_scale=-1.0), ValueError),
                        (dict(weights=torch.ones(2, device=DEV)), ValueError),
                        (dict(temperature=math.inf), ValueError)):
        with pytest.raises(err):
            ops.topk_distill_loss(x, ids, logq, **{**good, **change})
    with pytest.raises(ValueError):
        ops.topk_distill_loss(x, ids, logq[:, :3], denom=1.0)
    with pytest.raises(ValueError):
        ops.topk_distill_loss(x, ids[:2], logq[:2], denom=1.0)
    with pytest.raises(TypeError):
        ops.topk_distill_loss(x, ids.float(), logq, denom=1.0)
    with pytest.raises(ValueError):
        ops.topk_distill_loss(x, ids.repeat(1, 65), logq.repeat(1, 65), denom=1.0)
    with pytest.raises(ValueError):
        ops.fused_lm_head_topk_distill(x, torch.randn(7, 49, device=DEV), ids, logq, denom=1.0)


def test_vocabulary_beyond_the_kernels_is_refused():
    ops = _ops()
    x = torch.zeros(1, (1 << 22) + 1, device=DEV, dtype=torch.float16)
    with pytest.raises(ValueError, match="larger"):
        ops.token_logprobs(x)
    with pytest.raises(ValueError, match="larger"):
        ops.topk_distill_loss(x, torch.zeros(1, 1, dtype=torch.long, device=DEV), torch.zeros(1, 1, device=DEV),
                              denom=1.0)
    y = x[:, :1 << 22]
    y[0, 4000000] = 3.0
    r = ops.token_logprobs(y, None, top_k=2)
    assert r.top_ids.tolist() == [[4000000, 0]]
    _, rows = ops.topk_distill_loss(y, r.top_ids, r.top_logp, denom=1.0)
    assert abs(float(rows[0])) < 1e-5
