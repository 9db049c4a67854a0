"""Low-rank adapters of many requests at once, beside a shared projection.

A batch packs the rows of several requests; request ``i`` owns rows ``cu[i]:cu[i+1]`` and uses the adapter
in slot ``s_i`` of ``A [S, R, K]``, ``B [S, N, R]`` (``-1``: none, the shared weight alone -- a reference
policy next to the policies that are trained from it).  With ``W [N, K]`` and a factor ``c_s``::

    y_t  = W x_t + B_s u_t           u_t  = c_s A_s x_t
    dx_t = W^T dy_t + A_s^T du_t     du_t = c_s B_s^T dy_t
    dA_s = sum_t du_t x_t^T          dB_s = sum_t dy_t u_t^T          (t over the rows of slot s)

:func:`adapter_rows` lays out once per batch which rows use which slot; every projection of the model takes
the same plan.  On CUDA (``csrc/adapter_linear.cu``; BF16 or FP16, sums in FP32, ``u`` and ``du`` rounded to
the inputs' type for ``y`` and ``dx``, in two parts of it for ``dB`` and ``dA``) the low-rank products join the projection's own accumulators, whatever mix of slots a
tile of rows holds, and a row takes nothing from another request: an adapter that has gone to infinity or
NaN spoils its own rows and gradients only.  Results do not depend on timing.  On CPU, and as the library
baseline, the PyTorch form runs, in any floating type.

The rounding of ``u`` and ``du`` is one of range too.  In FP16 a value above 65504 makes its row of ``y`` (``dx``), and its
slot's ``dB`` (``dA``), infinite or NaN also where they would be finite themselves, never finite and wrong; and below 6e-5, as
``du`` is while ``B`` is still near zero, steps of 6e-8 are what is left of it: carry a loss scale that keeps ``B^T dy`` above that.
BF16 has FP32's range.

``K``, ``N`` and ``R`` are multiples of 8 on CUDA and ``R`` is at most 128; adapters of different ranks share a
stack by rows and columns of zeros.  A slot without rows has zero gradients.  A parameter's FP32
``main_grad`` (``A``, ``B`` and ``W`` alike) is added to in place of a returned gradient.  The gradient of ``W``
is BF16 only.  There is a first derivative only.
"""

from __future__ import annotations

from typing import Sequence

import numpy as np
import torch
from torch import Tensor

from ._ext import kernels, on_gpu, reference_forced
from .norm import _main_grad

MAX_RANK = 128
_TILE = 256       # rows of a tile whose slots the plan lists, and
_BLOCK = 64       # most rows of one slot that a gradient's sum takes at a time


class AdapterRows:
    """Which rows of a packed batch use which adapter slot (made by :func:`adapter_rows`)."""

    def __init__(self, cu_seqlens: list[int], slots: list[int], device: torch.device) -> None:
        self.cu_seqlens, self.slots = cu_seqlens, slots
        self.num_rows = cu_seqlens[-1]
        self.num_slots = max(slots, default=-1) + 1       # a stack needs at least as many
        if device.type == "cuda" and not reference_forced():
            self.table, self.meta = kernels().adapter_plan(cu_seqlens, slots, device)
        else:
            table, self.meta = _lay_out(cu_seqlens, slots)
            self.table = torch.from_numpy(table).to(device)
        self.device = self.table.device


def _lay_out(cu: list[int], slots: list[int]) -> tuple[np.ndarray, list[int]]:
    """The plan as the kernels read it (``csrc/adapter_ops.cpp`` lays out the same for them): one int32 buffer, and
    ``[rows, slots, units, blocks, where its parts begin]``.

    * ``row_slot [T]``;
    * per tile of 256 rows, the slots that it meets: ``tile_start [tiles + 1]`` into ``pairs [., 12]`` =
      (slot, 0, 0, 0, 8 words with the bits of the rows that are NOT the slot's);
    * the same by tiles of 128 rows, each pair by itself: ``unit_start [tiles + 1]`` into ``units [., 8]`` = (tile,
      slot, 0, 0, 4 words);
    * per slot, its rows in blocks of at most 64: ``block_start [slots + 1]`` into ``blocks [., 4]`` = (first
      row, rows, slot, 0).  A block ends where the slot's rows end, so that it holds no other request's row.
    """
    rows, top = cu[-1], max(slots, default=-1) + 1
    row_slot = np.repeat(np.asarray(slots, np.int64), np.diff(np.asarray(cu, np.int64)))
    at = np.flatnonzero(row_slot >= 0)
    tiles = -(-rows // _TILE)
    keys, pair = np.unique((at // _TILE) * max(top, 1) + row_slot[at], return_inverse=True)
    off = np.ones((len(keys), _TILE), np.uint8)
    off[pair, at % _TILE] = 0
    pairs = np.zeros((len(keys), 12), np.int32)
    pairs[:, 0] = keys % max(top, 1)
    pairs[:, 4:] = np.packbits(off, axis=1, bitorder="little").view(np.int32)
    halves = pairs[:, 4:].reshape(-1, 2, 4)
    pair, half = np.nonzero((halves != -1).any(axis=2))
    units = np.zeros((len(pair), 8), np.int32)
    units[:, 0], units[:, 1], units[:, 4:] = keys[pair] // max(top, 1) * 2 + half, pairs[pair, 0], halves[pair, half]
    units = units[np.argsort(units[:, 0], kind="stable")]
    unit_start = np.searchsorted(units[:, 0], np.arange(2 * tiles + 1))
    tile_start = np.searchsorted(keys // max(top, 1), np.arange(tiles + 1))

    first = np.flatnonzero(np.diff(row_slot, prepend=-2))            # runs of one slot, whatever their requests
    length = np.diff(np.append(first, rows))
    first, length = first[row_slot[first] >= 0], length[row_slot[first] >= 0]
    count = -(-length // _BLOCK)
    run = np.repeat(np.arange(len(first)), count)
    step = np.arange(len(run)) - np.repeat(np.cumsum(count) - count, count)
    row = first[run] + _BLOCK * step
    owner = row_slot[row]
    blocks = np.stack((row, np.minimum(_BLOCK, length[run] - _BLOCK * step), owner, 0 * row), axis=1)
    order = np.argsort(owner, kind="stable")
    block_start = np.searchsorted(owner[order], np.arange(top + 1))

    parts, where, total = [], [], 0
    for part in (row_slot, tile_start, pairs, unit_start, units, block_start, blocks[order]):
        flat = np.asarray(part, np.int32).reshape(-1)
        where.append(total)
        parts.append(np.concatenate((flat, np.zeros(-len(flat) % 4, np.int32))))      # each begins at 16 bytes
        total += len(parts[-1])
    return np.concatenate(parts), [rows, top, len(units), len(blocks), *where]


def adapter_rows(cu_seqlens: Sequence[int], slots: Sequence[int], device=None) -> AdapterRows:
    """The plan of a packed batch: request ``i`` has rows ``cu_seqlens[i]:cu_seqlens[i+1]`` and slot ``slots[i]`` (-1: none).

    Both are host lists; ``device`` is where the batch lives (the current CUDA device unless given, else the CPU).
    Requests may be empty, share slots, and come in any order.  One plan serves any number of calls, on any streams, and may
    be let go after the last one; with a CUDA graph it is made before the capture and kept as long as the graph.  Its
    copy to the device is waited for, behind what the current stream has under way."""
    cu, slots = list(map(int, cu_seqlens)), list(map(int, slots))
    if len(cu) != len(slots) + 1 or cu[0] != 0 or any(b < a for a, b in zip(cu, cu[1:])):
        raise ValueError(f"adapter_rows: cu_seqlens must rise from 0 and have one entry more than the {len(slots)} slots")
    if any(s < -1 for s in slots):
        raise ValueError(f"adapter_rows: a slot is -1 (no adapter) or counts from 0, got {min(slots)}")
    if cu[-1] >= 1 << 30 or max(slots, default=-1) >= 1 << 16:
        raise ValueError("adapter_rows: at most 2^30 rows and 2^16 slots")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else "cpu"
    device = torch.device(device)
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adapter_rows: a plan cannot be made while a CUDA graph is captured; make it before")
    return AdapterRows(cu, slots, device)


def adapter_linear_reference(x: Tensor, weight: Tensor, a: Tensor, b: Tensor, rows: AdapterRows,
                             scale: Tensor | float = 1.0) -> Tensor:
    """PyTorch form: FP32 (or wider) products of the inputs as they are, one rounding at the end."""
    wide = torch.promote_types(x.dtype, torch.float32)
    xf, af, bf = x.to(wide), a.to(wide), b.to(wide)
    y = xf @ weight.to(wide).t()
    parts = []
    for lo, hi, s in zip(rows.cu_seqlens, rows.cu_seqlens[1:], rows.slots):
        part = y[lo:hi]
        if s >= 0 and hi > lo:
            part = part + (scale[s] if isinstance(scale, Tensor) else scale) * ((xf[lo:hi] @ af[s].t()) @ bf[s].t())
        parts.append(part)
    # (every stack stays in the graph, so that a slot without rows has a gradient of zeros)
    y = torch.cat(parts) if parts else y
    return (y + 0.0 * (af[:, :0].sum() + bf[:, :0].sum())).to(x.dtype)


def _check(x, weight, a, b, rows, scale) -> None:
    for name, t, dims in (("x", x, 2), ("weight", weight, 2), ("a", a, 3), ("b", b, 3)):
        if not isinstance(t, Tensor) or t.dim() < dims or (name != "x" and t.dim() != dims):
            raise ValueError(f"adapter_linear: {name} must be a tensor of {dims} dimensions")
        if not t.is_floating_point():
            raise TypeError(f"adapter_linear: {name} must be floating point, got {t.dtype}")
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError(f"adapter_linear: {name} is {t.dtype} on {t.device}, x {x.dtype} on {x.device}")
    k, (n, kw), (s, r, ka), (sb, nb, rb) = x.shape[-1], weight.shape, a.shape, b.shape
    if kw != k or ka != k or nb != n or sb != s or rb != r:
        raise ValueError(f"adapter_linear: x [.., {k}], weight {tuple(weight.shape)}, a {tuple(a.shape)} and "
                         f"b {tuple(b.shape)} do not fit [T, K], [N, K], [S, R, K], [S, N, R]")
    if not isinstance(rows, AdapterRows):
        raise TypeError("adapter_linear: rows must come from adapter_rows()")
    t = x.numel() // k if k else 0
    if rows.num_rows != t:
        raise ValueError(f"adapter_linear: the requests cover {rows.num_rows} rows but x has {t}")
    if rows.num_slots > s:
        raise ValueError(f"adapter_linear: a request uses slot {rows.num_slots - 1} of a stack of {s}")
    if rows.device != x.device:
        raise TypeError(f"adapter_linear: rows were laid out for {rows.device}, x is on {x.device}")
    if isinstance(scale, Tensor) and (scale.shape != (s,) or scale.device != x.device or scale.requires_grad
                                      or not scale.is_floating_point()):
        raise ValueError(f"adapter_linear: scale must be a number or one per slot [{s}] on {x.device}, without gradient")


def _check_cuda(x, weight, a) -> None:
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"adapter_linear: bfloat16 or float16 on CUDA, got {x.dtype}")
    s, r, k = a.shape
    if s < 1 or k < 8 or k % 8 or weight.shape[0] < 8 or weight.shape[0] % 8:
        raise ValueError(f"adapter_linear: K ({k}) and N ({weight.shape[0]}) must be multiples of 8, and the stack must "
                         "not be empty")
    if r < 8 or r % 8 or r > MAX_RANK:
        raise ValueError(f"adapter_linear: rank {r} must be a multiple of 8 up to {MAX_RANK} (smaller ones: pad with zeros)")
    if weight.requires_grad and x.dtype == torch.float16:
        raise ValueError("adapter_linear: the shared weight's gradient is BF16 only; freeze the FP16 weight")


def _plain(t: Tensor, rows: bool) -> Tensor:
    """``t`` with unit columns, rows 16 bytes apart or a multiple, and an aligned address; a copy where it is not."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() or (rows and t.stride(-1) == 1 and t.stride(0) % 8 == 0
                                                         and t.stride(0) >= t.shape[1])):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def adapter_linear(x: Tensor, weight: Tensor, a: Tensor, b: Tensor, rows: AdapterRows,
                   scale: Tensor | float = 1.0) -> Tensor:
    """``y_t = W x_t + scale_s B_s (A_s x_t)`` for the rows ``x [.., K]`` of a batch that ``rows`` describes.

    ``weight [N, K]``, ``a [S, R, K]``, ``b [S, N, R]``; ``scale`` is a number or FP32 ``[S]`` (no gradient).
    Differentiable in ``x``, ``weight``, ``a`` and ``b``."""
    if not on_gpu(x):
        _check(x, weight, a, b, rows, scale)
        y = adapter_linear_reference(x.reshape(-1, x.shape[-1]), weight, a, b, rows, scale)
        return y.view(*x.shape[:-1], weight.shape[0])
    mains = tuple(None if not p.requires_grad else _stacked(_main_grad(p), p) for p in (a, b, weight))
    per_slot = isinstance(scale, Tensor)
    run = kernels().adapter_linear
    if isinstance(rows, AdapterRows):
        y = run(x, weight, a, b, rows.table, rows.meta, 1.0 if per_slot else scale, scale if per_slot else None, *mains)
        if y is not None:
            return y
    _check(x, weight, a, b, rows, scale)
    _check_cuda(x, weight, a)
    if per_slot:
        scale = scale.float().contiguous()
    x2 = _plain(x.reshape(-1, x.shape[-1]), True)
    y = run(x2, _plain(weight, True), _plain(a, False), _plain(b, False), rows.table, rows.meta,
            1.0 if per_slot else scale, scale if per_slot else None, *mains)
    if y is None:
        raise ValueError("adapter_linear: sizes out of range (2^30 rows or columns, 2^16 slots)")
    return y.view(*x.shape[:-1], weight.shape[0])


def _stacked(main: Tensor | None, p: Tensor) -> Tensor | None:
    """An accumulator that the kernels can add to; autograd returns the gradient where there is none."""
    return None if main is None or main.numel() != p.numel() or main.data_ptr() % 16 else main.view(p.shape)
