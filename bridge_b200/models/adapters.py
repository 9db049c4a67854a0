"""Low-rank adapters on a frozen policy model: several policies at once over one set of weights.

:class:`AdapterSet` holds, for every adapted projection of a model, the stacks ``A [S, R, K]`` and ``B [S, N, R]`` of
``S`` slots (policies), freezes the model, and hooks itself into the projections.  Inside :meth:`AdapterSet.use` the
model's forward takes each row through its request's slot; outside of it the model is the reference policy it was::

    adapters = AdapterSet(model, slots=8, rank=16)
    optimizer = MixedPrecisionAdamW(adapters, AdamWConfig(grad_clip=0.0))
    with adapters.use(adapter_rows(cu_seqlens, slots)):
        hidden = model(ids, positions)
        ...
        loss.backward()                            # inside, where activations are computed again
    norms = adapters.clip_grad_norm_(1.0)          # each policy by its own norm
    optimizer.step()

``B`` begins at zero, so that a fresh slot is the reference policy.

With an engine: ``forward_backward_batch`` inside ``use(slot)`` gives one slot's gradients (its executors take a batch apart,
so a plan of several requests does not fit their rows); over data-parallel ranks the caller adds them up.  ``train_step`` and
``optimizer_step``, which step the model's own weights, are refused.
"""

from __future__ import annotations

import contextlib
import math
import warnings

import torch
import torch.nn as nn
from torch import Tensor

from ..ops.adapter import MAX_RANK, AdapterRows, adapter_linear, adapter_rows
from ..ops.grad_norm import clip_grad_norm
from ..parallel.tp import ColumnParallelLinear, RowParallelLinear, tp_size
from .moe import MoELayer

TARGETS = ("qkv", "o_proj", "in_proj", "out_proj", "fc1", "fc2")


class _Adapted:
    """What an adapted projection calls in place of its product (no submodule of it: the model keeps its parameters)."""

    def __init__(self, owner: "AdapterSet", a: nn.Parameter, b: nn.Parameter) -> None:
        self.owner, self.a, self.b = owner, a, b

    def __call__(self, x: Tensor, weight: Tensor) -> Tensor | None:
        rows = self.owner.rows_for(x)
        return None if rows is None else adapter_linear(x, weight, self.a, self.b, rows, self.owner.scale)


class AdapterSet(nn.Module):
    """Adapters of ``slots`` policies on the ``targets`` projections of ``model`` (unsharded; its weights are frozen).

    ``scale`` is ``alpha / rank`` (``alpha`` is the rank unless given).  The experts of mixture-of-experts layers, routed and
    shared, get no adapters; a warning says so where ``targets`` name MLP projections."""

    def __init__(self, model: nn.Module, *, slots: int, rank: int, alpha: float | None = None,
                 targets: tuple[str, ...] = TARGETS, seed: int = 0) -> None:
        super().__init__()
        if slots < 1 or rank < 1:
            raise ValueError(f"AdapterSet: needs at least one slot and rank 1, got {slots} and {rank}")
        found = [(name, m) for name, m in model.named_modules()
                 if isinstance(m, (ColumnParallelLinear, RowParallelLinear)) and name.rsplit(".", 1)[-1] in targets]
        if not found:
            raise ValueError(f"AdapterSet: the model has no projection named one of {targets}")
        if any(tp_size(m.group) > 1 for _, m in found):
            raise NotImplementedError("AdapterSet: tensor-parallel projections are not adapted")
        if any(m.weight.is_cuda for _, m in found) and (rank % 8 or rank > MAX_RANK):
            raise ValueError(f"AdapterSet: on CUDA the rank is a multiple of 8 up to {MAX_RANK}, got {rank}")
        if any(m.adapter is not None for _, m in found):
            raise ValueError("AdapterSet: the model has adapters already; remove() them first")
        experts = [name for name, m in model.named_modules() if isinstance(m, MoELayer)]
        if experts and {"fc1", "fc2"} & set(targets):
            warnings.warn(f"AdapterSet: the routed and shared experts of {len(experts)} mixture-of-experts layers get no "
                          f"adapters ({experts[0]} the first)", stacklevel=2)
        self.slots, self.rank, self.scale = slots, rank, (rank if alpha is None else alpha) / rank
        self.active: AdapterRows | int | None = None
        self._open = 0              # use() blocks under way
        self._used = False          # whether one of them had adapters
        self._plans: dict[tuple[int, int, str], AdapterRows] = {}
        self._captured: dict[tuple[int, int, str], AdapterRows] = {}     # those that a CUDA graph may read again
        self._modules_of = [m for _, m in found]        # (a list: the model's modules do not become this one's)
        g = torch.Generator().manual_seed(seed)
        self.a, self.b = nn.ParameterDict(), nn.ParameterDict()
        for name, m in found:
            (n, k), w = m.weight.shape, m.weight
            key = name.replace(".", "/")
            a = torch.randn(slots, rank, k, generator=g) / math.sqrt(k)
            self.a[key] = nn.Parameter(a.to(device=w.device, dtype=w.dtype))
            self.b[key] = nn.Parameter(torch.zeros(slots, n, rank, device=w.device, dtype=w.dtype))
            m.adapter = _Adapted(self, self.a[key], self.b[key])
        model.requires_grad_(False)

    def remove(self) -> None:
        """Take the adapters off the model (its weights stay frozen)."""
        for m in self._modules_of:
            m.adapter = None

    @contextlib.contextmanager
    def use(self, rows: AdapterRows | int | None):
        """Forwards inside run ``rows``' requests through their slots; an integer: every row through that slot;
        ``None``: the model as it was.  One setting at a time, for all threads.

        A forward that a backward pass computes again (activation checkpointing) takes the setting of that moment, so the
        backward belongs inside the block of its forward.  Outside of every block it is refused rather than taken
        through the model without its adapters."""
        if isinstance(rows, int) and not -1 <= rows < self.slots:
            raise ValueError(f"AdapterSet: slot {rows} of {self.slots}")
        if not (rows is None or isinstance(rows, (int, AdapterRows))):
            raise TypeError("AdapterSet: use() takes adapter_rows(), a slot or None")
        before, self.active = self.active, rows
        self._open += 1
        self._used = self._used or rows is not None
        try:
            yield self
        finally:
            self._open -= 1
            self.active = before

    def rows_for(self, x: Tensor) -> AdapterRows | None:
        """The plan of a projection's input, or None for the model as it was."""
        if self.active is None and self._used and not self._open and torch._C._current_graph_task_id() != -1:
            raise RuntimeError("AdapterSet: a backward pass computes a forward again outside of use(); run the backward inside "
                               "the block of its forward (use(None) for the model as it was)")
        if not isinstance(self.active, int):
            return self.active
        if self.active < 0:
            return None
        t = x.numel() // x.shape[-1]
        key = (t, self.active, str(x.device))
        plan = self._plans.get(key) or self._captured.get(key)
        if plan is None:
            if len(self._plans) >= 256:
                self._plans.clear()
            plan = self._plans[key] = adapter_rows([0, t], [self.active], device=x.device)
        if x.is_cuda:
            with torch.cuda.device(x.device):
                if torch.cuda.is_current_stream_capturing():
                    self._captured[key] = plan
        return plan

    def gradients(self) -> list[Tensor]:
        """The stacks' gradients (FP32 ``main_grad`` where an optimizer keeps one), of those that have any."""
        grads = [getattr(p, "main_grad", None) if getattr(p, "main_grad", None) is not None else p.grad
                 for p in self.parameters()]
        return [g for g in grads if g is not None]

    def clip_grad_norm_(self, max_norm: Tensor | float, *, grad_scale: float = 1.0) -> Tensor:
        """Clip each slot's gradients by their own norm, in place; the norms from before, ``[S]``."""
        grads = self.gradients()
        if not grads:
            raise ValueError("AdapterSet: no gradients to clip")
        return clip_grad_norm(grads, max_norm, per_slot=True, grad_scale=grad_scale)
