"""Adapters beside a shared projection where a pair of SMs takes tile after tile: against 64 bits (bounds: adapter_oracle)."""

import pytest
import torch

from bridge_b200.ops import adapter_linear, adapter_rows
from test_adapter_gpu import DEV, _compare, _inputs

pytestmark = pytest.mark.gpu


def _mixed(t):
    """Requests whose ends fall inside tiles, of slots 0 to 2 and of none."""
    ends = sorted({1, t // 7, t // 3, t // 2 + 5, t - 130, t - 1, t})
    return [0] + ends, [(i + 1) % 4 - 1 for i in range(len(ends))]


# A last tile of columns with 1 to 64 or 129 to 192 of its 256 has an odd number of stores of 64; another whole tile of the
# same pair follows it.  K is one or two steps, so that the next tile's sums are ready while the stores still go out.
@pytest.mark.parametrize("t,k,n,dtype", [(16384, 64, 320, torch.bfloat16), (16384, 64, 264, torch.float16),
                                         (16384, 64, 392, torch.bfloat16), (16384, 64, 448, torch.bfloat16),
                                         (20000, 128, 64, torch.bfloat16), (20000, 64, 128, torch.float16),
                                         (4700, 128, 12352, torch.bfloat16), (5000, 136, 1216, torch.bfloat16)])
def test_odd_numbers_of_stores(t, k, n, dtype):
    x, w, a, b, dy = _inputs(t, k, n, 3, 16, dtype, seed=t + n)
    cu, slots = _mixed(t)
    got = _compare(x, w, a, b, cu, slots, [2.0, 0.5, -1.0], dy)
    rows, scale = adapter_rows(cu, slots, device=DEV), torch.tensor([2.0, 0.5, -1.0], device=DEV)
    for _ in range(10):
        with torch.no_grad():
            assert torch.equal(adapter_linear(x, w, a, b, rows, scale), got["y"])


# Forward and backward: 16 of 90 tiles cut in four, both ways; 6 of 80, and 8 of 304, in eight; none, and 32 of 180 in two;
# none (49 columns of tiles in groups of 16 rows), and all 24 in three.
@pytest.mark.parametrize("t,k,n,dtype", [(2100, 2560, 2560, torch.bfloat16), (2047, 9728, 2560, torch.float16),
                                         (4600, 2560, 5888, torch.bfloat16), (517, 2048, 12352, torch.bfloat16)])
def test_rounds_of_tiles_cut_along_k(t, k, n, dtype):
    x, w, a, b, dy = _inputs(t, k, n, 3, 24, dtype, seed=t + n)
    cu, slots = _mixed(t)
    _compare(x, w, a, b, cu, slots, [2.0, 0.5, -1.0], dy)


def test_wide_last_column_at_full_size():
    """A hybrid model's input projection."""
    t, k, n = 8192, 2048, 12352
    x, w, a, b, dy = _inputs(t, k, n, 3, 8, torch.bfloat16)
    cu, slots = _mixed(t)
    _compare(x, w, a, b, cu, slots, 1.0, dy)
