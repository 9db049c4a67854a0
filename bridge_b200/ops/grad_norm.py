"""Norm over many gradient tensors, and clipping: of all together, or of each slot of stacked gradients.

Stacked gradients (``[S, ...]``, as those of :func:`~bridge_b200.ops.adapter.adapter_linear`'s ``A`` and ``B``) belong to
``S`` trainings that know nothing of each other; with ``per_slot`` each is clipped by its own norm::

    norm_s = sqrt(sum over tensors and values of g_s^2) / grad_scale
    out_s  = g_s min(1, max_norm / (norm_s + 1e-6)) / grad_scale

``grad_scale`` is the loss scale that the gradients carry.  The norm is the one of
:class:`~bridge_b200.engine.optim.MixedPrecisionAdamW`; its sum and the factor are 64-bit, so that finite gradients are
scaled right whatever their size (the norm itself is returned in FP32, infinite above 3.4e38).  A NaN or infinite gradient
makes the norm NaN or infinite and, times the factor (NaN or 0), its slot's gradients NaN where they were not finite.
Subnormal FP32 gradients count as 0 on CUDA, and so do FP32 results that would be subnormal.  Results do not depend on timing
(``csrc/grad_norm.cu``); on CPU the PyTorch form runs.  Nothing here is differentiable.
"""

from __future__ import annotations

import math
from typing import Sequence

import torch
from torch import Tensor

from ._ext import kernels, on_gpu


def _check(grads, grad_scale: float) -> list[Tensor]:
    if not isinstance(grads, (list, tuple)):
        grads = list(grads)
    if not grads or not isinstance(grads[0], Tensor):
        raise ValueError("clip_grad_norm: needs a list of gradient tensors, without None")
    if not (grad_scale > 0 and math.isfinite(grad_scale)):
        raise ValueError(f"clip_grad_norm: grad_scale must be positive and finite, got {grad_scale}")
    return grads


def _tensors(*lists) -> None:
    """(The binding looks at every entry by itself: on CUDA this only finds the words for what it refused.)"""
    for entries in lists:
        if any(not isinstance(t, Tensor) for t in entries):
            raise ValueError("clip_grad_norm: needs lists of tensors, without None")


def _run(*args):
    try:
        return kernels().clip_grad_norm(*args)
    except TypeError:
        _tensors(args[0], args[-1])
        raise


def _detached(tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("clip_grad_norm: norms and clipped gradients are not differentiable; detach the tensors")


def _groups(g: Tensor, per_slot: bool, slots: int) -> Tensor:
    if per_slot and (g.dim() == 0 or g.shape[0] != slots):
        raise ValueError(f"clip_grad_norm: gradients are stacks of {slots} slots, got one of sizes {list(g.shape)}")
    return g.reshape(slots, -1)


def clip_grad_norm_reference(grads: list[Tensor], max_norm, per_slot: bool, grad_scale: float, out) -> Tensor:
    """PyTorch form."""
    slots = (grads[0].shape[0] if grads[0].dim() else 0) if per_slot else 1
    if per_slot and slots < 1:
        raise ValueError("clip_grad_norm: per_slot needs gradients stacked by slot")
    total = torch.zeros(slots, dtype=torch.float64, device=grads[0].device)
    for g in grads:
        if not g.is_floating_point():
            raise TypeError(f"clip_grad_norm: gradients are floating point, got {g.dtype}")
        total = total + _groups(g, per_slot, slots).double().square().sum(dim=1)
    norm = total.sqrt() / grad_scale
    if out is not None:
        bound = max_norm.double().reshape(-1) if isinstance(max_norm, Tensor) else torch.full_like(norm, max_norm)
        factor = torch.where(norm + 1e-6 <= bound, torch.ones_like(norm), bound / (norm + 1e-6)) / grad_scale
        for g, o in zip(grads, out):
            o.copy_((_groups(g, per_slot, slots).double() * factor[:, None]).view(g.shape))
    return norm.float() if per_slot else norm.float()[0]


def global_grad_norm(grads: Sequence[Tensor], *, per_slot: bool = False, grad_scale: float = 1.0) -> Tensor:
    """2-norm over all tensors, FP32 ``[]``; with ``per_slot`` ``[S]``, each slot's own.  No host synchronisation."""
    grads = _check(grads, grad_scale)
    if on_gpu(grads[0]):
        return _run(grads, per_slot, grad_scale, False, 0.0, None, [])
    _tensors(grads)
    _detached(grads)
    with torch.no_grad():
        return clip_grad_norm_reference(grads, 0.0, per_slot, grad_scale, None)


def clip_grad_norm(grads: Sequence[Tensor], max_norm: Tensor | float, *, per_slot: bool = False, grad_scale: float = 1.0,
                   out: Sequence[Tensor] | None = None) -> Tensor:
    """Scale gradients down to ``max_norm`` and return the norm from before, as :func:`global_grad_norm` does.

    The gradients (dense FP32, BF16 or FP16 tensors of any mix, on one device) are overwritten, or left and written to
    ``out``, tensors like them that may be FP32.  ``max_norm`` is a number, or FP32 ``[S]`` with ``per_slot``."""
    grads = _check(grads, grad_scale)
    if out is not None and not isinstance(out, (list, tuple)):
        out = list(out)
    if out is not None and len(out) != len(grads):
        raise ValueError(f"clip_grad_norm: one output per gradient, got {len(out)} for {len(grads)}")
    out = [] if out is None else out
    bounds = isinstance(max_norm, Tensor)
    if not bounds and not max_norm >= 0:
        raise ValueError(f"clip_grad_norm: max_norm must not be negative, got {max_norm}")
    if on_gpu(grads[0]):
        return _run(grads, per_slot, grad_scale, True, 0.0 if bounds else max_norm, max_norm if bounds else None, out)
    _tensors(grads, out)
    _detached([*grads, *out])
    with torch.no_grad():
        return clip_grad_norm_reference(grads, max_norm, per_slot, grad_scale, out or grads)
