"""Adapters under activation checkpointing: the forward that a backward pass computes again has to see the same slots."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from bridge_b200.models import AdapterSet, build_model, get_config
from bridge_b200.ops import adapter_rows


def _setup():
    model = build_model(get_config("tiny"), seed=1, dtype=torch.float32)
    adapters = AdapterSet(model, slots=2, rank=8, seed=3)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for p in adapters.b.values():
            p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    # (two projections of a layer in a row)
    layer = adapters._modules_of[-2:]
    x = torch.randn(9, layer[0].weight.shape[1], generator=g, requires_grad=True)

    def forward(x):
        y = layer[0](x)
        return layer[1](torch.tanh(y[:, :layer[1].weight.shape[1]]))

    return adapters, forward, x


def _gradients(adapters, x, y, backward=None):
    for p in (x, *adapters.parameters()):
        p.grad = None
    (backward or (lambda: y.square().sum().backward()))()
    return [None if p.grad is None else p.grad.clone() for p in (x, *adapters.parameters())]


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("setting", ["rows", 1])
def test_recomputed_inside_the_block(reentrant, setting):
    adapters, forward, x = _setup()
    rows = adapter_rows([0, 4, 5, 9], [1, -1, 0], device="cpu") if setting == "rows" else setting
    with adapters.use(rows):
        want = _gradients(adapters, x, forward(x))
        got = _gradients(adapters, x, checkpoint(forward, x, use_reentrant=reentrant))
    assert sum(g is not None for g in want) == 5
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_outside_of_every_block_is_refused(reentrant):
    adapters, forward, x = _setup()
    with adapters.use(1):
        y = checkpoint(forward, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="inside the block"):
        y.square().sum().backward()


def test_model_as_it_was_is_recomputed_where_that_is_said():
    adapters, forward, x = _setup()
    want = _gradients(adapters, x, forward(x))
    got = _gradients(adapters, x, checkpoint(forward, x, use_reentrant=False))       # no adapters in use yet
    assert torch.equal(got[0], want[0])
    with adapters.use(1), torch.no_grad():
        forward(x)
    with adapters.use(None):
        got = _gradients(adapters, x, checkpoint(forward, x, use_reentrant=False))
    assert torch.equal(got[0], want[0])
    # a backward that computes no forward again may come later
    with adapters.use(0):
        y = forward(x)
    _gradients(adapters, x, y)
    assert any(p.grad is not None for p in adapters.parameters())
