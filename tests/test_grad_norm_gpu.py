"""Norm and clipping of many gradients on the GPU, against 64 bits.

Bounds: squares are summed in FP32 by eights and in 64 bits from there on, so the sum of squares is off by 8 half steps
``2^-24`` at most and the norm by 4, plus its rounding; a scaled value by the norm's 4, the factor's and the product's
rounding, and half a step of its own type (below FP16's normal numbers 2^-25).
"""

import math

import pytest
import torch

from bridge_b200.ops import clip_grad_norm, global_grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2.0 ** -24


def _want(grads, bound, slots, grad_scale):
    groups = [g.double().reshape(slots, -1) for g in grads]
    norm = sum((g * g).sum(1) for g in groups).sqrt() / grad_scale
    bound = torch.as_tensor(bound, dtype=torch.float64, device=DEV).expand(slots)
    factor = torch.where(norm + 1e-6 <= bound, torch.ones_like(norm), bound / (norm + 1e-6)) / grad_scale
    return norm, [(g * factor[:, None]).view(x.shape) for g, x in zip(groups, grads)]


def _check(grads, bound, *, per_slot=False, grad_scale=1.0, out_type=None, at=None):
    slots = grads[0].shape[0] if per_slot else 1
    given = bound.float() if isinstance(bound, torch.Tensor) else bound
    norm, scaled = _want(grads, given, slots, grad_scale)
    alone = global_grad_norm(grads, per_slot=per_slot, grad_scale=grad_scale)
    out = None
    if out_type is not None:
        out = [torch.empty_like(g, dtype=out_type) for g in grads]
        kept = [g.clone() for g in grads]
    got = clip_grad_norm(grads, given, per_slot=per_slot, grad_scale=grad_scale, out=out)
    assert got.shape == ((slots,) if per_slot else ()) and torch.equal(got, alone)
    assert ((got.double().reshape(-1) - norm).abs() <= 5 * STEP * norm).all()
    for o, w in zip(out or grads, scaled):
        half = torch.finfo(o.dtype).eps / 2
        tiny = 2.0 ** -25 if o.dtype == torch.float16 else 2.0 ** -126
        assert ((o.double() - w).abs() <= (6 * STEP + half) * w.abs() + tiny).all()
    if out is not None:
        assert all(torch.equal(g, k) for g, k in zip(grads, kept))
    return got


def _grads(shapes, dtype, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(s, device=DEV, generator=g).mul_(std).to(dtype) for s in shapes]


SHAPES = [(1,), (7,), (33, 5), (2048,), (2049,), (3, 1111), (256, 129), (0,), (64, 64), (1000, 77)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bound", [1e-2, 5.0, math.inf])
@pytest.mark.parametrize("more", [[], [(700, 1001)], [(3000, 2003), (5, 1 << 20), (7,)]])
def test_types_and_sizes(dtype, bound, more):
    """Lists below and above 1 MB, and beyond 2^24 values."""
    for out_type in (None, dtype, torch.float32):
        _check(_grads(SHAPES + more, dtype), bound, out_type=out_type, grad_scale=1.0 if out_type is None else 64.0)


def test_mixed_types_in_one_list():
    grads = _grads(SHAPES[:4], torch.float32) + _grads(SHAPES[4:7], torch.bfloat16) + _grads(SHAPES[7:], torch.float16)
    _check(grads, 3.0, out_type=torch.float32)
    _check(grads, 3.0)


@pytest.mark.parametrize("slots,more", [(1, 0), (3, 0), (17, 0), (32, 0), (33, 0), (5, 130001), (200, 3001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_by_slot(slots, more, dtype):
    """Odd sizes, so that the slots begin at any alignment; one slot is clipped, one is not, one is zero."""
    grads = _grads([(slots, 3, 5), (slots, 2191), (slots, 1), (slots, 29, 65), (slots, more)], dtype)
    for g in grads:
        g[0] *= 0.01
        g[-1] = 0 if slots > 1 else g[-1]
    got = _check(grads, 20.0, per_slot=True)
    if slots > 2:
        assert got[-1] == 0 and got[0] < 20.0 < got[1]
    _check(grads, torch.linspace(0.5, 40.0, slots, device=DEV), per_slot=True, grad_scale=8.0, out_type=torch.float32)


def test_many_tensors():
    """More than one launch takes, in place and with outputs that lie apart from their gradients."""
    shapes = [(17 + i % 301,) for i in range(1500)]
    flat = torch.randn(sum(s[0] for s in shapes), device=DEV)
    grads = list(flat.split([s[0] for s in shapes]))
    _check(grads, 2.0)
    _check(grads[::-1], 1.0, out_type=torch.float32)


def test_offsets_beyond_32_bits():
    n = (1 << 31) + 12345
    g = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g[0], g[1 << 30], g[-1] = 3.0, 4.0, 12.0
    norm = clip_grad_norm([g], 6.5)
    assert norm == 13.0
    assert (g[0], g[1 << 30], g[-1]) == (1.5, 2.0, 6.0) and int((g != 0).sum()) == 3


def test_large_and_small_values():
    """Squares outside FP32, next to ordinary ones."""
    for std in (1e25, 1e-25, 1e-30):
        _check(_grads([(1000,), (37,)], torch.float32, std=std), 1e-27 if std < 1 else 1.0, out_type=torch.float32)
    mixed = torch.randn(5000, device=DEV)
    mixed[::7] *= 1e22
    mixed[::11] *= 1e-22
    _check([mixed], 5.0)
    assert global_grad_norm([torch.zeros(100, device=DEV)]) == 0


def test_not_finite():
    grads = _grads([(3, 500), (3, 9)], torch.float32)
    grads[0][1, 7], grads[1][2, 3] = math.nan, -math.inf
    kept = [g.clone() for g in grads]
    norm = clip_grad_norm(grads, 1.0, per_slot=True)
    assert torch.isfinite(norm[0]) and torch.isnan(norm[1]) and norm[2] == math.inf
    assert all(torch.isfinite(g[0]).all() and torch.isnan(g[1]).all() for g in grads)
    assert torch.isnan(grads[1][2, 3]) and (grads[0][2] == 0).all()
    norm = clip_grad_norm(kept, math.inf, per_slot=True)         # nothing to clip
    assert norm[2] == math.inf and kept[1][2, 3] == -math.inf and torch.isfinite(kept[0][2]).all()


def test_layouts():
    base = torch.randn(64, 96, device=DEV)
    turned = base.clone().t()
    _check([turned, base.clone()], 2.0)
    _check([base.clone().t()], 2.0, out_type=torch.float32)
    flat = torch.randn(1001, device=DEV)
    _check([flat[1:8], flat[8:500], flat[501:]], 1.0)
    assert torch.equal(global_grad_norm([flat[:10], flat[5:15]]), global_grad_norm([flat[5:15], flat[:10]]))


def test_same_again_on_another_stream_and_captured():
    grads = _grads([(4, 999), (4, 64, 64)], torch.bfloat16)
    out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    want = clip_grad_norm(grads, 3.0, per_slot=True, out=out).clone()
    kept = [o.clone() for o in out]
    graphs, norms, outs = [], [], []
    for _ in range(2):
        into = [torch.zeros_like(o) for o in out]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grad_norm(grads, 3.0, per_slot=True, out=into))
        graphs.append(g)
        outs.append(into)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for norm, into in zip(norms, outs):
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(into, kept))


def test_in_place_is_seen_by_autograd():
    g = torch.randn(100, device=DEV)
    before = g._version
    clip_grad_norm([g], 1.0)
    assert g._version > before


def test_inference_tensors():
    with torch.inference_mode():
        g = torch.randn(100, device=DEV)
        before = g.clone()
        norm = clip_grad_norm([g], 1.0)
        assert torch.allclose(g, before / (norm + 1e-6), rtol=2 ** -21, atol=0)     # (three roundings here, two there)
        before = g.clone()
    assert global_grad_norm([g]) == global_grad_norm([before])
    with pytest.raises(RuntimeError, match="inference"):
        clip_grad_norm([g], 0.5)
    assert torch.equal(g, before)
    clip_grad_norm([g], 0.5, out=[torch.empty(100, device=DEV)])


def test_refusals():
    g = torch.randn(8, 16, device=DEV)
    for bad in ([g, None], [g, 1.0], [None, g]):
        with pytest.raises(ValueError, match="without None"):
            global_grad_norm(bad)
    with pytest.raises(ValueError, match="without None"):
        clip_grad_norm([g, g.clone()], 1.0, out=[g, None])
    assert torch.equal(global_grad_norm(x for x in (g, g)), global_grad_norm((g, g)))
    with pytest.raises(RuntimeError, match="differentiable"):
        global_grad_norm([g, g.clone().requires_grad_()])
    with torch.no_grad():
        assert global_grad_norm([g.clone().requires_grad_()]) == global_grad_norm([g])
    with pytest.raises(TypeError, match="float32"):
        global_grad_norm([g.double()])
    with pytest.raises(TypeError, match="cpu"):
        global_grad_norm([g, g.cpu()])
    with pytest.raises(ValueError, match="dense"):
        global_grad_norm([g[:, :3]])
    with pytest.raises(ValueError, match="dense"):
        global_grad_norm([g.t()], per_slot=True)
    with pytest.raises(ValueError, match="stacks of 8"):
        global_grad_norm([g, g[:4]], per_slot=True)
    with pytest.raises(ValueError, match="stacked by slot"):
        global_grad_norm([torch.ones((), device=DEV)], per_slot=True)
    for grads, out in (([g, g], None), ([g, g.view(-1)[8:]], None), ([g, g.clone()], [torch.empty_like(g)] * 2),
                       ([g[:4], g[4:]], [g[4:], g[:4]]), ([g.bfloat16()] * 2, [g, g])):
        with pytest.raises(ValueError, match="shares memory"):
            clip_grad_norm(grads, 1.0, out=out)
    with pytest.raises(TypeError, match="output"):
        clip_grad_norm([g], 1.0, out=[g.half()])
    with pytest.raises(ValueError, match="sizes"):
        clip_grad_norm([g], 1.0, out=[torch.empty(16, 8, device=DEV)])
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm([g], torch.ones(3, device=DEV), per_slot=True)
