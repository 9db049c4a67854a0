"""dA and dB are rounded to the inputs' type and, but for FP32's sums, nowhere else on the way from x, dy, A and B."""

import pytest
import torch

from adapter_oracle import half_step, row_slots
from bridge_b200.ops import adapter_rows
from test_adapter_gpu import DEV, _inputs, _train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,n,r", [(1, 264, 200, 16), (3, 2048, 2560, 8), (20, 512, 640, 32), (33, 512, 264, 64), (90, 256, 512, 128),
                                     (400, 640, 256, 24), (1500, 512, 1024, 72)])
def test_gradients_are_rounded_once(t, k, n, r, dtype):
    """Bound: half a step of the result; of u (du) in two parts 2^-16 relative in BF16 (2^-22 in FP16) of every product, with
    FP16's smallest step; and the FP32 sums of K (N) and of the rows, 2^-23 of what has been summed for each addition."""
    x, w, a, b, dy = _inputs(t, k, n, 2, r, dtype, seed=t + r)
    cu, slots, c = [0, (t + 1) // 2, t], [1, 0], 1.5
    got = _train(x, w, a, b, adapter_rows(cu, slots, device=DEV), c, dy)
    h, step, tiny = half_step(dtype), 2.0 ** -23, 2.0 ** -25 if dtype == torch.float16 else 0.0
    two = h * h
    x, a, b, dy = (v.double() for v in (x, a, b, dy))
    at = row_slots(cu, slots, DEV)
    for s in range(2):
        rows = at == s
        xs, ds = x[rows], dy[rows]
        u, du = c * xs @ a[s].t(), c * ds @ b[s]
        u_sum, du_sum = c * xs.abs() @ a[s].abs().t(), c * ds.abs() @ b[s].abs()
        m = int(rows.sum())
        for name, left, mid, mid_sum, length in (("da", xs, du, du_sum, n), ("db", ds, u, u_sum, k)):
            want = mid.t() @ left if name == "da" else left.t() @ mid
            off = (two + 2 * m * step) * mid.abs() + length * step * mid_sum + tiny
            bound = off.t() @ left.abs() if name == "da" else left.abs().t() @ off
            err = (got[name][s].double() - want).abs()
            assert (err <= h * want.abs() + bound + tiny).all(), (name, (err / (h * want.abs() + bound + tiny)).max())
        # and over all values the result's own rounding is what is left: uniform in half a step, 1 / sqrt(3) of it at most
        for name, want in (("da", du.t() @ xs), ("db", ds.t() @ u)):
            if m:
                assert (got[name][s].double() - want).norm() <= (0.6 * h + 2e-6) * want.norm(), name
