"""Adapters beside a shared projection in 64 bits, and how far rounding may take a result from it.

Bounds, element by element, with ``h`` half a step of the type (``eps / 2``) and FP32 sums of ``n`` products, each of
whose additions may drop up to one step ``2^-23`` of what has been summed:

* ``y = W x + B u``: ``h |y|`` (the result) + ``h |B| |u|`` (``u`` is rounded to the type) + ``2^-23 (K + R) (|W| |x| + |B| |u|)``
  and, inside ``u``, ``2^-23 K`` of ``c |B| |A| |x|``;
* ``dA = sum du x``: ``h |dA|`` + ``h sum |du| |x|`` + ``2^-23 (T sum |du| |x| + N c sum (|B| |dy|) |x|)``; ``dB`` likewise.
"""

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def row_slots(cu, slots, device):
    out = torch.full((cu[-1],), -1, dtype=torch.long, device=device)
    for a, b, s in zip(cu, cu[1:], slots):
        out[a:b] = s
    return out


def oracle(x, w, a, b, cu, slots, scale, dy=None):
    """``{name: (value, bound)}`` in 64 bits; ``scale`` a number or a list per slot."""
    h, step = half_step(x.dtype), 2.0 ** -23
    x, w, a, b = (t.detach().double() for t in (x, w, a, b))
    (t, k), n, (s, r, _) = x.shape, w.shape[0], a.shape
    at = row_slots(cu, slots, x.device)
    y, y_abs = x @ w.t(), x.abs() @ w.abs().t()
    by = (k + r) * step * y_abs
    out = {}
    mids = {}
    for i in range(s):
        rows = torch.nonzero(at == i).flatten()
        c = scale[i] if isinstance(scale, (list, tuple)) else scale
        u = c * (x[rows] @ a[i].t())
        u_sum = abs(c) * (x[rows].abs() @ a[i].abs().t())
        mids[i] = (rows, c, u, u_sum)
        y[rows] += u @ b[i].t()
        low = u.abs() @ b[i].abs().t()
        by[rows] += (h + (k + r) * step) * low + k * step * (u_sum @ b[i].abs().t())
    tiny = torch.finfo(torch.float16).smallest_normal * h       # what FP16 loses below its normal numbers
    out["y"] = (y, by + h * y.abs() + tiny)
    if dy is None:
        return out
    dy = dy.double()
    dx, bx = dy @ w, (n + r) * step * (dy.abs() @ w.abs())
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    ba, bb = torch.full_like(a, tiny), torch.full_like(b, tiny)
    for i, (rows, c, u, u_sum) in mids.items():
        du = c * (dy[rows] @ b[i])
        du_sum = abs(c) * (dy[rows].abs() @ b[i].abs())
        dx[rows] += du @ a[i]
        low = du.abs() @ a[i].abs()
        bx[rows] += (h + (n + r) * step) * low + n * step * (du_sum @ a[i].abs())
        m = len(rows)
        da[i], db[i] = du.t() @ x[rows], dy[rows].t() @ u
        ba[i] += h * da[i].abs() + (h + m * step) * (du.abs().t() @ x[rows].abs()) + n * step * (du_sum.t() @ x[rows].abs())
        bb[i] += h * db[i].abs() + (h + m * step) * (dy[rows].abs().t() @ u.abs()) + k * step * (dy[rows].abs().t() @ u_sum)
        # u and du below FP16's normal numbers are rounded to multiples of a fixed step
        ba[i] += tiny * x[rows].abs().sum(0)
        bb[i] += tiny * dy[rows].abs().sum(0)[:, None]
    out.update(dx=(dx, bx + h * dx.abs() + tiny * (1 + a.abs().sum(1).amax(0))), da=(da, ba), db=(db, bb))
    out["y"] = (out["y"][0], out["y"][1] + tiny * b.abs().sum(2).amax(0))
    return out


def assert_close(got, want, name):
    value, bound = want
    err = (got.detach().double() - value).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all(), name
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"
