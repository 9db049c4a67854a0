"""Norm and clipping of many gradients on the CPU."""

import math

import pytest
import torch

from bridge_b200.ops import clip_grad_norm, global_grad_norm


def test_all_together_and_by_slot():
    g = torch.Generator().manual_seed(0)
    grads = [torch.randn(3, 4, 5, generator=g), torch.randn(3, 7, generator=g), torch.randn(3, generator=g)]
    flat = torch.cat([x.flatten() for x in grads]).double()
    assert torch.allclose(global_grad_norm(grads, grad_scale=4.0).double(), flat.norm() / 4)
    by_slot = torch.stack([torch.cat([x[s].flatten() for x in grads]).norm() for s in range(3)])
    assert torch.allclose(global_grad_norm(grads, per_slot=True), by_slot)
    bound = by_slot.clone()
    bound[1] /= 2
    kept = [x.clone() for x in grads]
    norm = clip_grad_norm(grads, bound + 1e-3, per_slot=True)
    assert torch.allclose(norm, by_slot)
    for x, k in zip(grads, kept):
        assert torch.equal(x[0], k[0]) and torch.equal(x[2], k[2])
        assert torch.allclose(x[1], k[1] * (bound[1] + 1e-3) / (by_slot[1] + 1e-6))
    out = [torch.empty_like(x) for x in kept]
    clip_grad_norm(kept, math.inf, grad_scale=2.0, out=out)
    assert all(torch.equal(o, k / 2) for o, k in zip(out, kept))


def test_refusals():
    g = torch.ones(4)
    for bad in ([], [None], [g, None]):
        with pytest.raises(ValueError):
            global_grad_norm(bad)
    with pytest.raises(ValueError, match="grad_scale"):
        global_grad_norm([g], grad_scale=0.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm([g], -1.0)
    with pytest.raises(ValueError, match="stacks of 4"):
        global_grad_norm([g, torch.ones(3)], per_slot=True)
    with pytest.raises(ValueError, match="one output"):
        clip_grad_norm([g], 1.0, out=[])
    with pytest.raises(RuntimeError, match="differentiable"):
        global_grad_norm([g.clone().requires_grad_()])
