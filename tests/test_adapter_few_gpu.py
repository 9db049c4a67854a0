"""Gradients of a few rows: the same, to the bit, whatever others are asked for (the single-kernel form included)."""

import pytest
import torch

from bridge_b200.ops import adapter_rows
from test_adapter_gpu import DEV, _compare, _inputs, _train
from bridge_b200.ops import adapter_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,k,n,r", [(1, 4096, 2560, 16), (4, 4096, 2560, 16), (1, 2560, 6144, 16), (3, 6144, 2560, 16),
                                     (1, 4096, 4096, 64), (8, 2048, 8192, 8), (7, 8192, 2048, 8), (2, 264, 5000, 24)])
@pytest.mark.parametrize("slots", [[0, 0], [1, -1]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_only_what_is_asked_for(t, k, n, r, slots, dtype):
    x, w, a, b, dy = _inputs(t, k, n, 2, r, dtype, seed=t + k)
    cu = [0, (t + 1) // 2, t]
    rows = adapter_rows(cu, slots, device=DEV)
    want = _compare(x, w, a, b, cu, slots, 0.5, dy)
    for names in (("dx",), ("da",), ("db",), ("dx", "da"), ("dx", "db"), ("da", "db")):
        leaves = {"dx": x, "da": a, "db": b}
        live = {i: leaves[i].detach().requires_grad_() for i in names}
        y = adapter_linear(live.get("dx", x), w, live.get("da", a), live.get("db", b), rows, 0.5)
        for i, g in zip(names, torch.autograd.grad(y, [live[i] for i in names], dy)):
            assert torch.equal(g, want[i]), (i, names)


def test_a_run_of_steps_of_one_row():
    """Calls that begin while the ones before them end: a chain of them is what each gives by itself."""
    x, w, a, b, dy = _inputs(1, 2048, 2048, 2, 16, torch.bfloat16)
    rows = adapter_rows([0, 1], [1], device=DEV)
    alone = _train(x, w, a, b, rows, 1.0, dy)
    torch.cuda.synchronize()
    for _ in range(30):
        got = _train(x, w, a, b, rows, 1.0, dy)
        assert all(torch.equal(got[i], v) for i, v in alone.items())
