"""Distillation from a teacher that is known by its top log-probs.

Per row, a teacher gives ``K`` token ids with log-probs ``log q_j`` (a negative id drops the entry); the
student has ``p = softmax(x / T)`` over the whole vocabulary.  The divergence is

* ``tail=True``: ``KL(q || p)`` over the given tokens and ONE class of all others,
  ``sum_j q_j (log q_j - log p_j) + q_r (log q_r - log p_r)``, ``q_r = max(0, 1 - sum_j q_j)``;
* ``tail=False``: ``KL(q' || p)`` with ``q' = q / sum q`` (so raw top logits do as well).

With ``Q = sum_j q_j + q_r`` its gradient is ``dz_v = Q p_v - q_v`` on the given tokens and
``(Q - q_r / p_r) p_v`` elsewhere; ``loss = sum_u w_u KL_u / denom``.

The gradient of every row is known as soon as its statistics are, so the forward writes it
(``csrc/vocab_rows.cu``): the logits are read from memory once and the gradient is written once.  The
backward only checks that the loss was scaled by ``grad_scale`` as announced, and rescales otherwise (FP16
gradients are written again from the logits, which they keep for that: scaling what was rounded at another
scale would lose it).  Vocabularies in shards write theirs in the backward.
:func:`fused_lm_head_topk_distill` goes on to the LM head's own backward inside the forward and keeps what a
factor that only the backward knows is still to come to: a forward that is run again, or never followed by a
backward, changes no gradient.

Rows of weight 0 and rows without an entry have divergence 0 and gradient 0 whatever their logits hold.
A given token (``q_j > 0``) without student probability makes the divergence infinite, and so does a
tail without any; but a ``q_r`` of at most ``2^-18`` is then taken for the rounding of FP32 log-probs and
dropped (a teacher's alternatives under a mask that leaves no more than ``K`` tokens).
"""

from __future__ import annotations

import math

import torch
import torch.distributed as dist
from torch import Tensor

from ._ext import kernels, on_gpu
from .gemm import gemm
from .token_logprob import (MAX_TOP, _FLOOR, _LN2, _MASKED, check_ids, check_logits, check_shard, first_order,
                            join_shards, log2_scale, picked, row_floats, shard_sums, split_temperature, tp_world, unit_columns)


_RESIDUE = 2.0 ** -18      # of a teacher's probability that FP32 log-probs may leave by rounding


# ------------------------------------------------------------------------- PyTorch form (CPU, oracle)
def _open_reference(logits, ids, temp, temp1, vocab_start):
    """``(R, s)`` of the columns outside the given ids and the given ids' log2-domain logits, of one shard."""
    xc = logits.to(torch.promote_types(logits.dtype, torch.float32)) * log2_scale(temp, temp1, logits)
    given = _given(ids, vocab_start, xc)
    r, s, _ = shard_sums(torch.where(given, torch.full_like(xc, -math.inf), xc))
    return torch.stack((r, s), dim=1), picked(xc, ids, vocab_start).clamp(min=_MASKED)


def _given(ids, vocab_start, like):
    local = ids - vocab_start
    here = (local >= 0) & (local < like.shape[1])
    cols = torch.where(here, local, torch.full_like(local, like.shape[1]))
    given = torch.zeros((like.shape[0], like.shape[1] + 1), dtype=torch.bool, device=like.device)
    return given.scatter_(1, cols, True)[:, :-1]


def _finish_reference(stats, xc, ids, logq, weights, temp, temp1, scale, tail, total):
    """Rows, the factor of ``2^(xc - R)`` outside the given ids, and the given ids' gradients (64 bits inside)."""
    stats, xc, logq = stats.double(), xc.double(), logq.double()
    valid = (ids >= 0) & (ids < total)
    none = torch.full_like(logq, -math.inf)
    logq = torch.where(valid, logq, none)
    if not tail:
        norm = torch.logsumexp(logq, dim=1, keepdim=True)
        logq = torch.where(norm == -math.inf, none, logq - norm)
    q = torch.exp(logq)
    some = valid.any(dim=1)
    if not tail:
        some = some & (q.sum(dim=1) != 0)
    same = (ids[:, :, None] == ids[:, None, :]) & valid[:, :, None] & valid[:, None, :]
    first = valid & ~(torch.tril(same.int(), -1).bool().any(dim=2))
    share = (same * q[:, None, :]).sum(dim=2)                    # the id's probability, repeats together
    xc = torch.where(xc <= _MASKED, none, xc)
    r = torch.where(stats[:, 1] == 0, none[:, 0], stats[:, 0]) if logq.shape[1] else stats[:, 0]
    m = torch.maximum(r, torch.where(first, xc, none).amax(dim=1))
    lost = m <= _FLOOR                                           # no student probability anywhere
    m = torch.where(lost, torch.zeros_like(m), m)
    rest = torch.where(stats[:, 1] == 0, torch.zeros_like(m), stats[:, 1] * torch.exp2(r - m))
    z = torch.where(first, torch.exp2(xc - m[:, None]), torch.zeros_like(xc)).sum(dim=1) + rest
    log2z = torch.log2(z)
    logp = _LN2 * (xc - m[:, None] - log2z[:, None])
    kl = torch.where(q == 0, torch.zeros_like(q), q * (logq - logp)).sum(dim=1)
    q_rest = (1.0 - q.sum(dim=1)).clamp(min=0.0) if tail else torch.zeros_like(m)
    q_rest = torch.where((rest == 0) & (q_rest <= _RESIDUE), torch.zeros_like(m), q_rest)
    total_q = q.sum(dim=1) + q_rest
    p_rest = rest / z
    kl = kl + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - torch.log(p_rest)), torch.zeros_like(m))
    kl = torch.where(lost & ~torch.isnan(stats[:, 1]), torch.full_like(kl, math.inf), kl)
    w = torch.ones_like(m) if weights is None else weights.double()
    it = (1.0 / temp.double()) if temp is not None else torch.full_like(m, 1.0 / temp1)
    live = some & (w != 0) & ~lost
    f = torch.where(live, w * scale * it, torch.zeros_like(m))
    factor = torch.where(live & (stats[:, 1] != 0), f * (total_q * p_rest - q_rest) / stats[:, 1], torch.zeros_like(m))
    fix = torch.where(live[:, None], f[:, None] * (total_q[:, None] * torch.exp(logp) - share), torch.zeros_like(q))
    rows = torch.where(some & (w != 0), kl, torch.zeros_like(kl))
    return rows, torch.stack((stats[:, 0], factor), dim=1), torch.where(valid, fix, torch.zeros_like(fix))


def _grad_reference(logits, ids, coef, fix, temp, temp1, vocab_start, total):
    c = log2_scale(temp, temp1, logits)
    t = logits.to(c.dtype) * c - coef[:, :1].to(c.dtype)
    factor = coef[:, 1:].to(c.dtype)
    given = _given(ids, vocab_start, logits)
    g = torch.where(given | (factor == 0), torch.zeros_like(t), factor * torch.exp2(t))
    local = ids - vocab_start
    here = (ids >= 0) & (ids < total) & (local >= 0) & (local < logits.shape[1])
    rows, j = torch.nonzero(here, as_tuple=True)
    g[rows, local[rows, j]] = fix[rows, j].to(g.dtype)
    return g.to(logits.dtype)


# ------------------------------------------------------------------------------------------- one shard
def _rows(logits, ids, logq, weights, temp, temp1, scale, tail, vocab_start, group):
    """``(KL [U], coef, fix)`` of this rank's shard, in steps (and the PyTorch form)."""
    own, world = on_gpu(logits), tp_world(group)
    total = logits.shape[1] * world
    if own:
        stats, xc = kernels().distill_open(logits, ids, logq, weights, temp, temp1, vocab_start, total)
    else:
        stats, xc = _open_reference(logits, ids, temp, temp1, vocab_start)
    if world > 1:
        r, s = stats.unbind(1)
        r, s, _ = join_shards(r, s, torch.zeros_like(s), group)
        stats = torch.stack((r, s), dim=1)
        dist.all_reduce(xc, group=group)
    if own:
        return kernels().distill_finish(stats, xc, ids, logq, weights, temp, temp1, scale, tail, total)
    rows, coef, fix = _finish_reference(stats, xc, ids, logq, weights, temp, temp1, scale, tail, total)
    return rows.to(torch.promote_types(logits.dtype, torch.float32)), coef, fix


def _grad(logits, ids, coef, fix, temp, temp1, vocab_start, group, *, factor=None, inplace=False):
    """The shard's gradient, ``factor`` (on the device) times what the rows were finished for."""
    total = logits.shape[1] * tp_world(group)
    if factor is not None:
        coef, fix = torch.stack((coef[:, 0], coef[:, 1] * factor), dim=1), fix * factor
    if on_gpu(logits):
        return kernels().distill_grad(logits, ids, coef, fix, temp, temp1, vocab_start, total, inplace)
    return _grad_reference(logits, ids, coef, fix, temp, temp1, vocab_start, total)


def _weighted_sum(rows, weights, denom):
    if on_gpu(rows):
        return kernels().weighted_rows_sum(rows, weights, denom)
    if weights is None:
        return rows.sum() / denom
    return torch.where(weights != 0, rows * weights.to(rows.dtype), torch.zeros_like(rows)).sum() / denom


class _TopkDistillFn(torch.autograd.Function):
    """Vocabularies in shards, and the PyTorch form."""

    @staticmethod
    def forward(ctx, logits, ids, logq, weights, temp, temp1, tail, denom, grad_scale, vocab_start, group):
        rows, coef, fix = _rows(logits, ids, logq, weights, temp, temp1, grad_scale / denom, tail, vocab_start, group)
        ctx.save_for_backward(logits, ids, coef, fix, temp)
        ctx.at = temp1, vocab_start, group
        ctx.grad_scale = grad_scale
        ctx.mark_non_differentiable(rows)
        return _weighted_sum(rows, weights, denom), rows

    @staticmethod
    def backward(ctx, dloss, _drows):
        first_order("topk_distill_loss")
        logits, ids, coef, fix, temp = ctx.saved_tensors
        factor = dloss.to(coef.dtype) / ctx.grad_scale         # (before the one rounding to the logits' type)
        return (_grad(logits, ids, coef, fix, temp, *ctx.at, factor=factor),) + (None,) * 10


class _FusedHeadDistillFn(torch.autograd.Function):
    """LM head + divergence with the head's backward as far inside the forward as the loss's factor allows.

    ``dh`` is made in the forward and scaled in the backward.  For ``dW`` few rows keep their chunks'
    gradients, whose product with ``h`` the backward adds to ``main_grad`` itself; where these would be larger
    than an FP32 ``dW``, that is summed in the forward and added with the factor (4096 rows, H 2560, vocabulary
    151936, BF16, forward and backward: 8.6 to 8.8 ms kept as chunks, 9.7 to 10.7 ms summed).  FP16 heads do
    all of it in the backward, on the chunks' logits computed again: there only the loss's own factor says at
    which scale a gradient may be rounded."""

    @staticmethod
    def forward(ctx, h, weight, ids, logq, weights, temp, temp1, tail, denom, grad_scale, vocab_start, group,
                chunk_rows, differentiable):
        # (what needs a gradient is said of the inputs under no_grad too)
        want_dh, want_dw = (differentiable and n for n in ctx.needs_input_grad[:2])
        late = h.dtype == torch.float16 and (want_dh or want_dw)
        want = not late and (want_dh or want_dw)
        keep = want and want_dw and h.shape[0] * h.element_size() <= 4 * h.shape[1]
        dh, dw = _head_gradients(h, weight, want and want_dh, want and want_dw and not keep)
        parts, kept = [], []
        for at in _chunks(h, chunk_rows):
            lg = gemm(h[at], weight)
            teacher = (ids[at], logq[at], None if weights is None else weights[at], None if temp is None else temp[at],
                       temp1, grad_scale / denom, tail)
            if tp_world(group) == 1 and not late:
                parts.append((kernels().distill_rows_inplace(lg, *teacher, want), None, None))
                dlg = lg
            else:
                parts.append(_rows(lg, *teacher, vocab_start, group))
                if want:
                    dlg = _grad(lg, ids[at], *parts[-1][1:], *teacher[3:5], vocab_start, group, inplace=True)
            if want:
                _head_backward(dlg, h[at], weight, None if dh is None else dh[at], dw)
            if keep:
                kept.append(dlg)
        rows = torch.cat([p[0] for p in parts]) if parts else torch.zeros(0, dtype=torch.float32, device=h.device)
        ctx.late = (temp1, vocab_start, group) if late and parts else None
        if ctx.late:
            coef, fix = (torch.cat([p[i] for p in parts]) for i in (1, 2))
            ctx.save_for_backward(h, weight, ids, coef, fix, temp)
        else:
            ctx.save_for_backward(dh, dw, h if kept else None, *kept)
        ctx.grad_scale, ctx.chunk_rows, ctx.weight = grad_scale, chunk_rows, (weight.shape, weight.dtype)
        ctx.main_grad = getattr(weight, "main_grad", None)
        ctx.mark_non_differentiable(rows)
        return _weighted_sum(rows, weights, denom), rows

    @staticmethod
    def backward(ctx, dloss, _drows):
        first_order("fused_lm_head_topk_distill")
        f, main, (shape, dtype) = dloss.float() / ctx.grad_scale, ctx.main_grad, ctx.weight
        direct = main is not None and main.dtype == torch.float32      # a sum that products can be added to
        if ctx.late:
            h, weight, ids, coef, fix, temp = ctx.saved_tensors
            temp1, vocab_start, group = ctx.late
            dh, dw = _head_gradients(h, weight, ctx.needs_input_grad[0], ctx.needs_input_grad[1] and not direct)
            for at in _chunks(h, ctx.chunk_rows):
                dlg = _grad(gemm(h[at], weight), ids[at], coef[at], fix[at], None if temp is None else temp[at], temp1,
                            vocab_start, group, factor=f, inplace=True)
                _head_backward(dlg, h[at], weight, None if dh is None else dh[at],
                               main if direct and ctx.needs_input_grad[1] else dw)
            f = torch.ones_like(f)
        else:
            dh, dw, h, *kept = ctx.saved_tensors
            if dh is not None:
                dh = (dh.float() * f).to(dh.dtype)
            if kept:
                if not direct:
                    dw = torch.zeros(shape, dtype=torch.float32, device=h.device)
                hf = (h.float() * f).to(h.dtype)       # (rounded as dh is; exact for the announced factor)
                for at, dlg in zip(_chunks(h, ctx.chunk_rows), kept):
                    _head_backward(dlg, hf[at], None, None, main if direct else dw)
                f = torch.ones_like(f)
        if dw is not None and main is not None:
            main.addcmul_(dw.to(main.dtype), f.to(main.dtype))
            dw = None
        elif dw is not None:
            dw = (dw * f).to(dtype)
        return (dh, dw) + (None,) * 12


def _chunks(h, chunk_rows):
    return [slice(a, min(a + chunk_rows, h.shape[0])) for a in range(0, h.shape[0], chunk_rows)]


def _head_gradients(h, weight, want_dh, want_dw):
    return (torch.empty_like(h) if want_dh else None,
            torch.zeros(weight.shape, dtype=torch.float32, device=weight.device) if want_dw else None)


def _head_backward(dlg, h, weight, dh, dw):
    if dh is not None:
        dh.copy_(gemm(dlg, weight, b_mn=True))                         # dlogits @ W
    if dw is not None:
        gemm(dlg, h, a_mn=True, b_mn=True, out=dw, accumulate=True)    # += dlogits^T h


# ------------------------------------------------------------------------------------------------- API
def _arguments(name, rows, device, ids, logq, weights, temperature, denom, grad_scale):
    ids = check_ids(name, "teacher_ids", ids, rows, device)
    if ids.ndim != 2 or not 1 <= ids.shape[1] <= MAX_TOP:
        raise ValueError(f"{name}: teacher_ids must be [{rows}, K] with K in 1..{MAX_TOP}, got {tuple(ids.shape)}")
    if logq.shape != ids.shape:
        raise ValueError(f"{name}: teacher_logp must be {tuple(ids.shape)}, got {tuple(logq.shape)}")
    if logq.device != device or not logq.is_floating_point():
        raise ValueError(f"{name}: teacher_logp must be floating point on {device}")
    for what, v in (("denom", denom), ("grad_scale", grad_scale)):
        if not (float(v) > 0.0 and math.isfinite(float(v))):
            raise ValueError(f"{name}: {what} must be finite and positive, got {v!r}")
    if weights is not None:
        weights = row_floats(name, "weights", weights, rows, device)
    temp, temp1 = split_temperature(name, temperature, rows, device)
    if logq.dtype != torch.float32 or not logq.is_contiguous() or logq.requires_grad:
        logq = logq.detach().float().contiguous()
    return ids, logq, weights, temp, temp1


def topk_distill_loss(logits: Tensor, teacher_ids: Tensor, teacher_logp: Tensor, *, denom: float,
                      weights: Tensor | None = None, temperature: Tensor | float = 1.0, tail: bool = True,
                      grad_scale: float = 1.0, vocab_start: int = 0, tp_group=None) -> tuple[Tensor, Tensor]:
    """``(sum_u w_u KL_u / denom, KL [U])`` of a student's ``logits [U, V]``; only the loss is differentiable.

    ``teacher_ids`` / ``teacher_logp`` are ``[U, K]`` (``K`` up to 256; a negative id drops the entry, an id
    given twice counts as the sum of its probabilities in the gradient).  ``grad_scale`` announces the factor
    by which the caller multiplies the loss before ``backward`` (a loss scale); another one costs one more
    pass over the gradient, with one more rounding in BF16, or for FP16 logits the gradient once more.  ``backward``
    can be called once.  With ``tp_group``, ``logits`` is this rank's
    equal shard of the vocabulary and ``vocab_start`` its first token.
    """
    if tp_group is None and not vocab_start and on_gpu(logits):
        got = _own(logits, teacher_ids, teacher_logp, weights, temperature, tail, denom, grad_scale)
        if got:                                   # arguments that the kernels take as they are
            return got[0], got[1]
    name = "topk_distill_loss"
    check_logits(name, logits)
    check_shard(name, vocab_start, tp_group)
    args = _arguments(name, logits.shape[0], logits.device, teacher_ids, teacher_logp, weights, temperature, denom,
                      grad_scale)
    logits = unit_columns(logits)
    if tp_world(tp_group) == 1 and on_gpu(logits):
        got = kernels().topk_distill(logits, *args, tail, denom, grad_scale)
        if not got:
            raise ValueError(f"{name}: logits {tuple(logits.shape)} are larger than the kernels take")
        return got[0], got[1]
    return _TopkDistillFn.apply(logits, *args, tail, float(denom), float(grad_scale), vocab_start, tp_group)


def _own(logits, ids, logq, weights, temperature, tail, denom, grad_scale):
    try:
        if isinstance(temperature, Tensor):
            return kernels().topk_distill(logits, ids, logq, weights, temperature, 1.0, tail, denom, grad_scale)
        return kernels().topk_distill(logits, ids, logq, weights, None, temperature, tail, denom, grad_scale)
    except TypeError:                             # not even the right kinds of arguments: the checks say which
        return None


def fused_lm_head_topk_distill(h: Tensor, weight: Tensor, teacher_ids: Tensor, teacher_logp: Tensor, *, denom: float,
                               weights: Tensor | None = None, temperature: Tensor | float = 1.0, tail: bool = True,
                               grad_scale: float = 1.0, vocab_start: int = 0, tp_group=None,
                               chunk_rows: int = 4096) -> tuple[Tensor, Tensor]:
    """:func:`topk_distill_loss` of hidden rows ``h [U, H]`` under the head ``weight [V_local, H]``.

    The logits exist for ``chunk_rows`` rows at a time and become their own gradient in place.  Until the
    backward, which adds ``dW`` to ``weight.main_grad`` where there is one, these chunks are kept, or their sum
    ``dW`` in FP32, whichever is smaller; a ``grad_scale`` other than the loss's own factor costs ``dh`` and ``dW``
    one more rounding.  FP16 heads compute the logits once more in the backward instead.
    """
    name = "fused_lm_head_topk_distill"
    if h.ndim != 2 or weight.ndim != 2 or h.shape[1] != weight.shape[1]:
        raise ValueError(f"{name}: h {tuple(h.shape)} does not fit the head {tuple(weight.shape)}")
    if chunk_rows < 1:
        raise ValueError(f"{name}: chunk_rows must be positive")
    check_shard(name, vocab_start, tp_group)
    args = _arguments(name, h.shape[0], h.device, teacher_ids, teacher_logp, weights, temperature, denom, grad_scale)
    if on_gpu(h):
        return _FusedHeadDistillFn.apply(h.contiguous(), weight, *args, bool(tail), float(denom), float(grad_scale),
                                         int(vocab_start), tp_group, int(chunk_rows), torch.is_grad_enabled())
    return _TopkDistillFn.apply(torch.matmul(h, weight.t()), *args, bool(tail), float(denom), float(grad_scale),
                                int(vocab_start), tp_group)
