"""FP16 adapters whose low-rank values leave the type's range: seen in their own rows and gradients, and nowhere else."""

import pytest
import torch

from bridge_b200.ops import adapter_rows
from test_adapter_gpu import DEV, _inputs, _train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,r", [(3, 8), (40, 16), (100, 64), (400, 16)])
def test_above_the_largest_number(t, r):
    x, w, a, b, dy = _inputs(t, 512, 256, 2, r, torch.float16)
    cu, slots = [0, t // 3, t // 3 + 1, t], [0, 1, 0]
    rows = adapter_rows(cu, slots, device=DEV)
    row = t // 3
    others = [i for i in range(t) if i != row]
    clean = _train(x, w, a, b, rows, 1.0, dy)
    # u = 512 x 16 x 16 = 131072 where y takes 2^-9 of it
    big = {"x": x.clone(), "a": a.clone(), "b": b.clone()}
    big["x"][row], big["a"][1], big["b"][1] = 16.0, 16.0, 2.0 ** -9 / r
    got = _train(big["x"], w, big["a"], big["b"], rows, 1.0, dy)
    assert not torch.isfinite(got["y"][row]).any() and not torch.isfinite(got["db"][1]).any()
    assert torch.isfinite(got["da"]).all()
    for name in ("y", "dx"):
        assert torch.equal(got[name][others], clean[name][others])
    assert torch.equal(got["db"][0], clean["db"][0]) and torch.equal(got["da"][0], clean["da"][0])
    # du likewise
    big = {"b": b.clone(), "dy": dy.clone()}
    big["b"][1], big["dy"][row] = 32.0, 16.0
    got = _train(x, w, a, big["b"], rows, 1.0, big["dy"])
    assert not torch.isfinite(got["dx"][row]).any() and not torch.isfinite(got["da"][1]).any()
    assert torch.equal(got["dx"][others], clean["dx"][others])
    assert torch.equal(got["da"][0], clean["da"][0]) and torch.equal(got["db"][0], clean["db"][0])
