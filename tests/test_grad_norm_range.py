"""Clipping where the factor leaves FP32's range: finite gradients are scaled right whatever their size."""

import math

import pytest
import torch

from bridge_b200.ops import clip_grad_norm

STEP = 2.0 ** -24
# values, bound, grad_scale: factors of some 3e-42, 3e-41, 3e-46, 2e-39 and 1e39
CASES = [(1e25, 1e-15, 1.0), (1e36, 1e-3, 1.0), (1e36, 1e-8, 1.0), (1e30, 1.0, 2.0 ** 30), (1e-30, math.inf, 1e-39)]


def _run(device, std, bound, grad_scale, more, per_slot, out):
    g = torch.Generator().manual_seed(0)
    grads = [(torch.randn(s, generator=g, dtype=torch.float64) * std).float().to(device) for s in [(2, 501), (2, 7), (2, more)]]
    slots = 2 if per_slot else 1
    wide = [x.double().reshape(slots, -1) for x in grads]
    norm = sum((x * x).sum(1) for x in wide).sqrt() / grad_scale
    factor = (bound / (norm + 1e-6)).clamp(max=1.0) / grad_scale
    into = [torch.empty_like(x) for x in grads] if out else None
    got = clip_grad_norm(grads, bound, per_slot=per_slot, grad_scale=grad_scale, out=into)
    # (600 thousand values of 1e36 have a norm of 7.7e38, which is infinite in FP32)
    got, far = got.double().reshape(-1), norm > torch.finfo(torch.float32).max
    assert (got[far] == math.inf).all() and ((got - norm).abs()[~far] <= 5 * STEP * norm[~far]).all()
    for o, x in zip(into or grads, wide):
        want = (x * factor[:, None]).view(o.shape)
        # the norm's four half steps, the factor's and the product's; what is below FP32's normal numbers may be 0
        assert ((o.double() - want).abs() <= 7 * STEP * want.abs() + 2.0 ** -126).all()
        assert (o[want.abs() > 1e-37] != 0).all()


@pytest.mark.parametrize("std,bound,grad_scale", CASES)
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("out", [False, True])
def test_on_cpu(std, bound, grad_scale, per_slot, out):
    _run("cpu", std, bound, grad_scale, 33, per_slot, out)


@pytest.mark.gpu
@pytest.mark.parametrize("std,bound,grad_scale", CASES)
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("more", [33, 300001])
def test_on_gpu(std, bound, grad_scale, per_slot, out, more):
    """Lists below and above 1 MB."""
    _run("cuda", std, bound, grad_scale, more, per_slot, out)


def test_64_bit_gradients_on_cpu():
    g = torch.randn(1000, dtype=torch.float64)
    want = g / g.norm() * (g.norm() / (g.norm() + 1e-6))
    clip_grad_norm([g], 1.0)
    assert torch.allclose(g, want, rtol=1e-14, atol=0)


def test_norm_beyond_fp32():
    g = torch.full((4000,), 3e38)
    norm = clip_grad_norm([g], 1.0)
    assert norm == math.inf and torch.allclose(g, torch.full_like(g, 4000 ** -0.5))


@pytest.mark.gpu
def test_norm_beyond_fp32_on_gpu():
    for n in (4000, 400000):
        g = torch.full((n,), 3e38, device="cuda")
        norm = clip_grad_norm([g], 1.0)
        assert norm == math.inf and torch.allclose(g, torch.full_like(g, n ** -0.5))
