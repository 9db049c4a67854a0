"""Log-probs of given tokens with entropy and the likeliest alternatives, on rows of logits.

For logits ``x [U, V]`` and a temperature ``T`` per row, with ``z = x / T`` and ``p = softmax(z)``::

    logp[u, j]  = z[u, t_uj] - logsumexp(z[u])
    entropy[u]  = -sum_v p_v log p_v                                 (0 log 0 = 0)
    top[u]      = the k likeliest tokens, ties to the lower id, with their log-probs
    dx_v        = (sum_j g_j 1[v = t_j] - p_v sum_j g_j - dH p_v (log p_v + H)) / T

One pass over the logits forward, one read and one write backward (``csrc/vocab_rows.cu``); FP32, FP16
and BF16 rows of any stride and length.  :func:`fused_lm_head_token_logprobs` scores hidden rows, a chunk
of logits at a time; its alternatives are what :func:`~bridge_b200.ops.distill.topk_distill_loss` takes
as a teacher.

Edge cases: a token outside the vocabulary (a padded position) has log-prob 0 and no gradient.  A logit
of ``-inf``, or one with ``x / T`` at or below ``-2^31 ln 2`` (-1.49e9: FP32's lowest value, finite masks
from -1e10 down), carries no probability; where a row holds nothing else its log-probs are ``-inf``, its
entropy 0 and its gradient 0 (in other rows a finite fill has its own log-prob).  NaN, ``+inf`` or ``x / T`` above 1.49e9 in a row makes its log-probs and
entropy NaN (among the alternatives NaN counts as ``-inf``).  Subnormal logits count as 0.  There is a first derivative
only: a backward with ``create_graph=True`` and forward-mode inputs are refused.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.distributed as dist
from torch import Tensor

from ._ext import kernels, on_gpu
from .gemm import gemm

MAX_TOP = 256
_LN2 = math.log(2.0)
_LOG2E = 1.0 / _LN2
_FLOOR = -2.0 ** 31        # log2-domain logits at or below this carry no probability
_MASKED = -1e30            # ... and at or below this are as good as -inf
_FLOAT_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class TokenLogprobs(NamedTuple):
    """``None`` where not asked for.  ``logp`` and ``entropy`` are differentiable."""

    logp: Tensor | None         # [U] or [U, n], FP32
    entropy: Tensor | None      # [U], FP32
    top_ids: Tensor | None      # [U, k], int64, likeliest first
    top_logp: Tensor | None     # [U, k], FP32


# ------------------------------------------------------------------------------------------ arguments
def tp_world(group) -> int:
    return 1 if group is None else dist.get_world_size(group)


def check_shard(name: str, vocab_start: int, group) -> None:
    if vocab_start and tp_world(group) == 1:
        raise ValueError(f"{name}: vocab_start {vocab_start} says that this is a shard of the vocabulary, which needs "
                         "tp_group")


def check_logits(name: str, logits: Tensor) -> None:
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [U, V] with V >= 1, got {tuple(logits.shape)}")
    ok = _FLOAT_TYPES if logits.is_cuda else (*_FLOAT_TYPES, torch.float64)
    if logits.dtype not in ok:
        raise TypeError(f"{name}: logits must be float32, float16 or bfloat16, got {logits.dtype}")


def check_ids(name: str, what: str, ids: Tensor, rows: int, device) -> Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: {what} must be int64 or int32, got {ids.dtype}")
    if ids.ndim not in (1, 2) or ids.shape[0] != rows:
        raise ValueError(f"{name}: {what} must be [{rows}] or [{rows}, n], got {tuple(ids.shape)}")
    if ids.device != device:
        raise ValueError(f"{name}: {what} are on {ids.device}, the logits on {device}")
    return ids if ids.dtype == torch.int64 and ids.is_contiguous() else ids.long().contiguous()


def row_floats(name: str, what: str, value: Tensor, rows: int, device) -> Tensor:
    if value.shape != (rows,):
        raise ValueError(f"{name}: {what} must be [{rows}], got {tuple(value.shape)}")
    if value.device != device:
        raise ValueError(f"{name}: {what} is on {value.device}, the logits on {device}")
    if value.dtype == torch.float32 and value.is_contiguous() and not value.requires_grad:
        return value
    return value.detach().float().contiguous()


def split_temperature(name: str, temperature, rows: int, device) -> tuple[Tensor | None, float]:
    """``(per-row temperatures or None, the common one)``."""
    if isinstance(temperature, Tensor):
        return row_floats(name, "temperature", temperature, rows, device), 1.0
    t = float(temperature)
    if not (t > 0.0 and math.isfinite(t)):
        raise ValueError(f"{name}: temperature must be finite and positive, got {temperature!r}")
    return None, t


def unit_columns(logits: Tensor) -> Tensor:
    return logits if logits.shape[1] == 1 or logits.stride(1) == 1 else logits.contiguous()


# ------------------------------------------------------------------------- PyTorch form (CPU, oracle)
def log2_scale(temp: Tensor | None, temp1: float, logits: Tensor) -> Tensor:
    """``log2(e) / T`` per row, ``[U, 1]`` (broadcastable)."""
    dt = torch.promote_types(logits.dtype, torch.float32)
    if temp is None:
        return torch.full((1, 1), _LOG2E / temp1, dtype=dt, device=logits.device)
    return (_LOG2E / temp.to(dt))[:, None]


def _exact_scale(temp: Tensor | None, temp1: float, device, own: bool) -> Tensor:
    """:func:`log2_scale` in 64 bits; of the kernels, the FP32 number that they multiply by."""
    c = _LOG2E / (torch.full((1,), temp1, dtype=torch.float64, device=device) if temp is None else temp.double())
    return (c.float().double() if own else c)[:, None]


def shard_sums(xc: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """``(R, s, sum e t)`` of log2-domain rows: ``t = xc - R``, ``e = 2^t``; masked columns count nothing."""
    r = xc.amax(dim=1).clamp(min=_FLOOR)
    r = torch.where(r > -_FLOOR, torch.full_like(r, math.nan), r)
    t = torch.where(xc > _FLOOR, xc - r[:, None], torch.full_like(xc, -math.inf))
    t = torch.where(torch.isnan(xc), xc, t)
    e = torch.exp2(t)
    et = torch.where(e == 0, torch.zeros_like(e), e * t).sum(dim=1)
    return r, e.sum(dim=1), et


def join_shards(r: Tensor, s: Tensor, et: Tensor, group) -> tuple[Tensor, Tensor, Tensor]:
    """The sums of the whole vocabulary from every rank's ``(R, s, sum e t)`` (an all-reduce each of R and the sums)."""
    top = r.clone()
    dist.all_reduce(top, op=dist.ReduceOp.MAX, group=group)
    d = torch.where(s == 0, torch.zeros_like(r), r - top)
    k = torch.exp2(d)
    both = torch.stack((s * k, k * (et + d * s)))
    dist.all_reduce(both, group=group)
    return top, both[0], both[1]


def picked(xc: Tensor, ids: Tensor, vocab_start: int) -> Tensor:
    """``xc`` at the ids that this shard holds, 0 elsewhere."""
    local = ids - vocab_start
    here = (local >= 0) & (local < xc.shape[1])
    return torch.where(here, xc.gather(1, local.clamp(0, xc.shape[1] - 1)), torch.zeros((), dtype=xc.dtype,
                                                                                        device=xc.device))


def top_rows(x: Tensor, k: int) -> Tensor:
    """Columns of the ``k`` largest of every row, ties to the lower column; NaN counts as ``-inf``."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]


# -------------------------------------------------------------------------------------------- autograd
def first_order(name: str) -> None:
    """Called in a backward whose saved sums are constants: its result cannot be differentiated again."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no second derivative (backward was called with create_graph=True)")


class _TokenLogprobFn(torch.autograd.Function):
    """Vocabularies in shards, and the PyTorch form."""

    @staticmethod
    def forward(ctx, logits, tokens, temp, temp1, top_k, with_entropy, vocab_start, group):
        world = tp_world(group)
        total = logits.shape[1] * world
        own = on_gpu(logits)
        k = min(top_k, logits.shape[1])
        ctx.set_materialize_grads(False)
        ctx.vocab_start, ctx.total, ctx.temp1, ctx.own = vocab_start, total, temp1, own
        # Logits and sums travel as they are; what they make is worked out in 64 bits, like the kernel's own rows: a
        # log-prob is the small difference of x c and a log-sum that are as large as the logits.
        c = _exact_scale(temp, temp1, logits.device, own)
        out = torch.promote_types(logits.dtype, torch.float32)
        xt = picked(logits, tokens, vocab_start).to(out) if tokens is not None else None
        if own:
            _, sums, ids, top = kernels().token_logprob_open(logits, None, temp, temp1, k, with_entropy, vocab_start)
            r, s, et = sums.double().unbind(1)
        else:
            r, s, et = shard_sums(logits.double() * c)
            ids = top = None
            if k:
                ids = top_rows(logits, k)
                top = logits.gather(1, ids).to(out)
                ids = ids + vocab_start
        if world > 1:
            r, s, et = join_shards(r, s, et, group)
            if xt is not None:
                dist.all_reduce(xt, group=group)
            if top_k:
                ids, top = _join_tops(ids, top, top_k, world, group)
        log2s = torch.log2(s)
        full = r + log2s
        logp = None
        if tokens is not None:
            logp = _finish(xt.double() * c, full, s).to(out)
            logp = torch.where((tokens >= 0) & (tokens < total), logp, torch.zeros_like(logp))
        empty = s == 0
        one = torch.where(empty, torch.ones_like(s), s)
        ent = torch.where(empty, torch.zeros_like(s), _LN2 * (log2s - et / one)) if with_entropy else None
        stats = torch.stack((r, torch.where(empty, torch.zeros_like(s), 1.0 / one), et / one), dim=1)
        if own:
            stats = stats.float()
        if with_entropy:
            ent = ent.to(out)
        if top_k:
            top = _finish(top.double() * c, full, s).to(out)
            ctx.mark_non_differentiable(ids, top)
        ctx.save_for_backward(logits, tokens, temp, stats)
        return logp, ent, ids, top

    @staticmethod
    def backward(ctx, d_logp, d_ent, _ids, _top):
        first_order("token_logprobs")
        logits, tokens, temp, stats = ctx.saved_tensors
        if d_logp is None and d_ent is None:
            return (None,) * 8
        if ctx.own:
            f32 = [None if g is None else g.float().contiguous() for g in (d_logp, d_ent)]
            g = kernels().token_logprob_bwd(logits, tokens, temp, ctx.temp1, stats, f32[0], f32[1], ctx.vocab_start,
                                            ctx.total)
        else:
            g = _grad_reference(logits, tokens, temp, ctx.temp1, stats, d_logp, d_ent, ctx.vocab_start, ctx.total)
        return (g,) + (None,) * 7


def _finish(xc: Tensor, full: Tensor, s: Tensor) -> Tensor:
    """Log-probs of log2-domain logits under rows of log2-sum ``full``."""
    logp = _LN2 * (xc - full[:, None])
    gone = (xc <= _MASKED) | (s == 0)[:, None]
    return torch.where(gone, torch.full_like(logp, -math.inf), logp)


def _join_tops(ids: Tensor, top: Tensor, k: int, world: int, group) -> tuple[Tensor, Tensor]:
    """The ``k`` best of every rank's best.  Ranks hold ascending ids and equal logits are in id order within
    a rank, so the lower position of a tie is the lower id."""
    every_id = [torch.empty_like(ids) for _ in range(world)]
    every_top = [torch.empty_like(top) for _ in range(world)]
    dist.all_gather(every_id, ids.contiguous(), group=group)
    dist.all_gather(every_top, top.contiguous(), group=group)
    ids, top = torch.cat(every_id, dim=1), torch.cat(every_top, dim=1)
    if on_gpu(top):
        at = kernels().token_logprob_open(top, None, None, 1.0, k, False, 0)[2]
    else:
        at = top_rows(top, k)
    return ids.gather(1, at), top.gather(1, at)


def _grad_reference(logits, tokens, temp, temp1, stats, d_logp, d_ent, vocab_start, total):
    c = _exact_scale(temp, temp1, logits.device, False)
    r, inv, mean = (v[:, None] for v in stats.unbind(1))
    t = logits.double() * c - r
    p = torch.exp2(t) * inv
    g = torch.zeros_like(p)
    if d_logp is not None:
        held = (tokens >= 0) & (tokens < total)
        d = torch.where(held, d_logp.to(p.dtype), torch.zeros((), dtype=p.dtype, device=p.device))
        local = tokens - vocab_start
        here = held & (local >= 0) & (local < p.shape[1]) & (inv > 0)
        g = g - p * d.sum(dim=1, keepdim=True)
        g.scatter_add_(1, local.clamp(0, p.shape[1] - 1), torch.where(here, d, torch.zeros_like(d)))
    if d_ent is not None:
        g = g - torch.where(p == 0, torch.zeros_like(p), d_ent.to(p.dtype)[:, None] * p * (t - mean) * _LN2)
    return (g * (c * _LN2)).to(logits.dtype)


def token_logprobs(logits: Tensor, tokens: Tensor | None = None, temperature: Tensor | float = 1.0, *,
                   top_k: int = 0, with_entropy: bool = True, vocab_start: int = 0, tp_group=None) -> TokenLogprobs:
    """Log-probs of ``tokens`` (``[U]``, or ``[U, n]`` candidates a row) under ``softmax(logits / temperature)``.

    ``temperature`` is one positive number or ``[U]``; ``top_k`` (at most 256) also returns the likeliest
    tokens.  With ``tp_group``, ``logits`` is this rank's equal shard of the vocabulary, whose first token
    is ``vocab_start`` (0 without a group); every rank gets the whole result and its shard's gradient.
    """
    if tp_group is None and not vocab_start and on_gpu(logits):
        got = _own(logits, tokens, temperature, top_k, with_entropy)
        if got:                                   # arguments that the kernels take as they are
            return TokenLogprobs(*got)
    name = "token_logprobs"
    check_logits(name, logits)
    check_shard(name, vocab_start, tp_group)
    rows, device = logits.shape[0], logits.device
    world = tp_world(tp_group)
    total = logits.shape[1] * world
    if not 0 <= top_k <= min(MAX_TOP, total):
        raise ValueError(f"{name}: top_k must be within 0..{min(MAX_TOP, total)}, got {top_k}")
    if tokens is not None:
        tokens = check_ids(name, "tokens", tokens, rows, device)
    temp, temp1 = split_temperature(name, temperature, rows, device)
    logits = unit_columns(logits)
    if world == 1 and on_gpu(logits):
        got = kernels().token_logprobs(logits, tokens, temp, temp1, top_k, with_entropy)
        if not got:
            raise ValueError(f"{name}: logits {tuple(logits.shape)} are larger than the kernels take")
        return TokenLogprobs(*got)
    flat = tokens is not None and tokens.ndim == 1
    logp, ent, ids, top = _TokenLogprobFn.apply(logits, tokens[:, None] if flat else tokens, temp, temp1, top_k,
                                                with_entropy, vocab_start, tp_group)
    return TokenLogprobs(logp[:, 0] if flat else logp, ent, ids, top)


def _own(logits, tokens, temperature, top_k, with_entropy):
    try:
        if isinstance(temperature, Tensor):
            return kernels().token_logprobs(logits, tokens, temperature, 1.0, top_k, with_entropy)
        return kernels().token_logprobs(logits, tokens, None, temperature, top_k, with_entropy)
    except TypeError:                             # not even the right kinds of arguments: the checks say which
        return None


@torch.no_grad()
def fused_lm_head_token_logprobs(h: Tensor, weight: Tensor, tokens: Tensor | None = None,
                                 temperature: Tensor | float = 1.0, *, top_k: int = 0, with_entropy: bool = True,
                                 vocab_start: int = 0, tp_group=None, chunk_rows: int = 4096) -> TokenLogprobs:
    """:func:`token_logprobs` of hidden rows ``h [U, H]`` under the head ``weight [V_local, H]``, scoring only
    (no gradient): the logits exist for ``chunk_rows`` rows at a time."""
    name = "fused_lm_head_token_logprobs"
    if h.ndim != 2 or weight.ndim != 2 or h.shape[1] != weight.shape[1]:
        raise ValueError(f"{name}: h {tuple(h.shape)} does not fit the head {tuple(weight.shape)}")
    if chunk_rows < 1:
        raise ValueError(f"{name}: chunk_rows must be positive")
    if tokens is not None:
        tokens = check_ids(name, "tokens", tokens, h.shape[0], h.device)
    if isinstance(temperature, Tensor):
        temperature = row_floats(name, "temperature", temperature, h.shape[0], h.device)
    parts = []
    for a in range(0, max(h.shape[0], 1), chunk_rows):
        at = slice(a, min(a + chunk_rows, h.shape[0]))
        t = temperature[at] if isinstance(temperature, Tensor) else temperature
        parts.append(token_logprobs(gemm(h[at].contiguous(), weight), None if tokens is None else tokens[at], t,
                                    top_k=top_k, with_entropy=with_entropy, vocab_start=vocab_start,
                                    tp_group=tp_group))
    return TokenLogprobs(*(None if f[0] is None else torch.cat(f) for f in zip(*parts)))
