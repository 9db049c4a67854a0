"""Adapters beside a shared projection on the GPU, against 64 bits (bounds: adapter_oracle)."""

import math

import pytest
import torch

from adapter_oracle import assert_close, oracle
from bridge_b200.ops import adapter_linear, adapter_rows
from bridge_b200.ops._ext import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(t, k, n, s, r, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g).mul_(std).to(dtype)

    return (normal(t, k), normal(n, k, std=k ** -0.5), normal(s, r, k, std=k ** -0.5), normal(s, n, r, std=r ** -0.5),
            normal(t, n))


def _train(x, w, a, b, rows, scale, dy):
    x, a, b = (v.detach().requires_grad_() for v in (x, a, b))
    y = adapter_linear(x, w, a, b, rows, scale)
    return dict(zip(("y", "dx", "da", "db"), (y, *torch.autograd.grad(y, (x, a, b), dy))))


def _compare(x, w, a, b, cu, slots, scale, dy):
    rows = adapter_rows(cu, slots, device=DEV)
    per_slot = torch.tensor(scale, device=DEV) if isinstance(scale, list) else scale
    got = _train(x, w, a, b, rows, per_slot, dy)
    want = oracle(x, w, a, b, cu, slots, scale, dy)
    for name, v in want.items():
        assert_close(got[name], v, name)
    with torch.no_grad():
        assert torch.equal(adapter_linear(x, w, a, b, rows, per_slot), got["y"])
    assert kernels().adapter_error_code() == 0
    return got


# rows, requests' ends, slots
MIXES = [
    ([1], [0]),
    ([1], [-1]),
    ([2, 3], [1, 0]),
    ([7, 7, 16], [0, 2, 1]),
    ([63, 64], [-1, 1]),
    ([1, 2, 3, 4, 65], [2, 0, 2, -1, 1]),
    ([127, 128], [0, 0]),
    ([129], [2]),
    ([100, 200, 255], [0, 1, 0]),
    ([256, 257], [1, 2]),
    ([5, 300, 301, 512, 700], [0, 1, 2, -1, 0]),
    (list(range(1, 101)), [i % 4 - 1 for i in range(100)]),
    ([400, 1100], [-1, 2]),
]


@pytest.mark.parametrize("mix", range(len(MIXES)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_and_requests(mix, dtype):
    ends, slots = MIXES[mix]
    x, w, a, b, dy = _inputs(ends[-1], 264, 200, 3, 16, dtype, seed=mix)
    _compare(x, w, a, b, [0] + ends, slots, [2.0, 0.5, -1.0], dy)


@pytest.mark.parametrize("k,n,r", [(8, 8, 8), (16, 1032, 24), (72, 64, 40), (1032, 16, 8), (512, 256, 64), (520, 264, 72),
                                   (2560, 136, 128), (128, 2568, 96), (4104, 520, 16), (1000, 1000, 56)])
@pytest.mark.parametrize("t", [1, 5, 40, 70, 333])
def test_sizes(k, n, r, t):
    x, w, a, b, dy = _inputs(t, k, n, 4, r, torch.bfloat16, seed=k + n + r + t)
    cu = [0, t // 3, t // 2, t]
    _compare(x, w, a, b, cu, [3, 0, 1], 2.0, dy)


@pytest.mark.parametrize("t,n", [(3, 19456), (70, 19208), (128, 37000), (5, 40000)])
def test_more_columns_than_multiprocessors(t, n):
    """Few rows and tiles that are a few more than there are SMs."""
    x, w, a, b, dy = _inputs(t, 136, n, 3, 16, torch.bfloat16, seed=n)
    _compare(x, w, a, b, [0, t // 3, t - 1, t], [2, 0, -1], 1.0, dy)


@pytest.mark.parametrize("t", [9, 300, 2500])
def test_an_adapter_spoils_its_own_rows_only(t):
    """Infinite and NaN adapters, and rows that hold them, beside requests that share their tiles and blocks."""
    cu, slots = [0, t // 3, t // 2, t - 2, t], [0, 1, 2, 1]
    x, w, a, b, dy = _inputs(t, 264, 200, 3, 16, torch.bfloat16)
    rows = adapter_rows(cu, slots, device=DEV)
    clean = _train(x, w, a, b, rows, 1.0, dy)
    for at, fill in (("a", math.nan), ("b", math.inf), ("x", math.nan), ("dy", math.inf)):
        bad = {"x": x.clone(), "a": a.clone(), "b": b.clone(), "dy": dy.clone()}
        if at in ("a", "b"):
            bad[at][1] = fill
        else:
            bad[at][cu[1]:cu[2]] = fill
            bad[at][cu[3]:] = fill
        got = _train(bad["x"], w, bad["a"], bad["b"], rows, 1.0, bad["dy"])
        for lo, hi in ((cu[0], cu[1]), (cu[2], cu[3])):
            assert torch.equal(got["y"][lo:hi], clean["y"][lo:hi]), at
            assert torch.equal(got["dx"][lo:hi], clean["dx"][lo:hi]), at
        for s in (0, 2):
            assert torch.equal(got["da"][s], clean["da"][s]) and torch.equal(got["db"][s], clean["db"][s]), at
    assert not torch.isfinite(_train(x, w, a * math.nan, b, rows, 1.0, dy)["y"]).any()


@pytest.mark.parametrize("seed", range(12))
def test_plan_is_the_one_laid_out_without_cuda(seed):
    g = torch.Generator().manual_seed(seed)
    count = int(torch.randint(0, 60, (), generator=g))
    lengths = torch.randint(0, [3, 40, 900][seed % 3], (count,), generator=g).tolist()
    slots = torch.randint(-1, [1, 5, 40, 3][seed // 3], (count,), generator=g).tolist()
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    host, dev = adapter_rows(cu, slots, device="cpu"), adapter_rows(cu, slots, device=DEV)
    assert host.meta == list(dev.meta) and torch.equal(host.table, dev.table.cpu())


def test_no_adapter_is_the_projection():
    x, w, a, b, dy = _inputs(300, 256, 512, 2, 8, torch.bfloat16)
    got = _train(x, w, a * math.nan, b * math.inf, adapter_rows([0, 300], [-1], device=DEV), 1.0, dy)
    want = oracle(x, w, 0 * a, 0 * b, [0, 300], [-1], 1.0, dy)
    assert_close(got["y"], want["y"], "y")
    assert_close(got["dx"], want["dx"], "dx")
    assert got["da"].abs().sum() == 0 and got["db"].abs().sum() == 0


def test_no_rows_and_empty_requests():
    x, w, a, b, dy = _inputs(30, 64, 72, 5, 8, torch.bfloat16)
    _compare(x, w, a, b, [0, 0, 10, 10, 30, 30], [4, 0, 1, 3, 2], 1.0, dy)
    got = _train(x[:0], w, a, b, adapter_rows([0, 0], [3], device=DEV), 1.0, dy[:0])
    assert got["y"].shape == (0, 72) and got["dx"].shape == (0, 64)
    assert got["da"].abs().sum() == 0 and got["db"].abs().sum() == 0


@pytest.mark.parametrize("t", [12, 150])
def test_strides_and_alignment(t):
    """Slices of wider buffers, rows at odd offsets, transposed and broadcast inputs, batch dimensions."""
    x, w, a, b, dy = _inputs(t, 136, 128, 3, 24, torch.bfloat16)
    cu, slots = [0, 5, t], [2, 0]
    rows = adapter_rows(cu, slots, device=DEV)
    want = _train(x, w, a, b, rows, 1.5, dy)

    def check(x=x, w=w, a=a, b=b, dy=dy):
        got = _train(x, w, a, b, rows, 1.5, dy)
        for name, v in want.items():
            assert torch.equal(got[name], v), name

    wide = torch.randn(t, 400, device=DEV).to(torch.bfloat16)
    wide[:, 64:200] = x
    check(x=wide[:, 64:200])
    odd = torch.empty(t * 136 + 3, device=DEV, dtype=torch.bfloat16)[3:].view(t, 136)
    check(x=odd.copy_(x))
    check(x=x.t().contiguous().t(), w=w.t().contiguous().t(), dy=dy.t().contiguous().t())
    check(a=a.transpose(1, 2).contiguous().transpose(1, 2), b=b.transpose(0, 1).contiguous().transpose(0, 1))
    flat = torch.empty(a.numel() + 1, device=DEV, dtype=a.dtype)[1:].view(a.shape).copy_(a)
    check(a=flat)
    got = _train(x, w, a, b, rows, 1.5, torch.ones((), device=DEV, dtype=dy.dtype).expand(dy.shape))
    assert torch.equal(got["dx"], _train(x, w, a, b, rows, 1.5, torch.ones_like(dy))["dx"])
    y = adapter_linear(x.view(2, t // 2, 136), w, a, b, rows, 1.5)
    assert y.shape == (2, t // 2, 128) and torch.equal(y.view(t, 128), want["y"])
    one = adapter_rows([0, 1], [1], device=DEV)
    row = _train(x[3].expand(1, 136), w, a, b, one, 1.5, dy[3].expand(1, 128))
    assert_close(row["y"], oracle(x[3:4], w, a, b, [0, 1], [1], 1.5)["y"], "y")


@pytest.mark.parametrize("t", [20, 600])
def test_shared_weight_gradient_and_accumulators(t):
    x, w, a, b, dy = _inputs(t, 256, 512, 2, 16, torch.bfloat16)
    cu, slots = [0, t // 2, t], [1, 0]
    rows = adapter_rows(cu, slots, device=DEV)
    plain = _train(x, w, a, b, rows, 1.0, dy)
    x, w, a, b = (v.detach().requires_grad_() for v in (x, w, a, b))
    (dw,) = torch.autograd.grad(adapter_linear(x, w, a, b, rows), (w,), dy)
    want = dy.double().t() @ x.detach().double()
    # half a step of BF16 (8 significant bits, eps 2^-7) is 2^-8; the sum of t products as in the oracle
    bound = 2.0 ** -8 * want.abs() + t * 2.0 ** -23 * (dy.double().abs().t() @ x.detach().double().abs())
    assert ((dw.double() - want).abs() <= bound).all()
    for p in (w, a, b):
        p.main_grad = torch.ones(p.shape, device=DEV)
    for passes in (1, 2):
        adapter_linear(x, w, a, b, rows).backward(dy)
        assert w.grad is None and a.grad is None and b.grad is None
        full = oracle(x, w, a, b, cu, slots, 1.0, dy)
        for p, name in ((a, "da"), (b, "db")):
            value, bound = full[name]
            assert_close(p.main_grad, (1 + passes * value, passes * bound + 2.0 ** -20), name)
        assert ((w.main_grad.double() - 1 - passes * want).abs() <= passes * (t * 2.0 ** -22 + 2.0 ** -20) * (
            1 + dy.double().abs().t() @ x.detach().double().abs())).all()
    assert torch.equal(x.grad, plain["dx"] + plain["dx"])


@pytest.mark.parametrize("t,k,n", [(300, 256, 512), (1660, 176, 2936), (913, 4424, 656), (22, 2168, 2400)])
def test_only_what_is_asked_for(t, k, n):
    """A gradient is the same, to the bit, whatever others are asked for."""
    x, w, a, b, dy = _inputs(t, k, n, 2, 16, torch.bfloat16)
    rows = adapter_rows([0, t // 3, t], [1, 0], device=DEV)
    want = _train(x, w, a, b, rows, 1.0, dy)
    for name, v in (("dx", x), ("da", a), ("db", b)):
        leaf = v.detach().requires_grad_()
        args = [leaf if t is v else t for t in (x, w, a, b)]
        (g,) = torch.autograd.grad(adapter_linear(*args, rows), (leaf,), dy)
        assert torch.equal(g, want[name]), name


@pytest.mark.parametrize("t", [17, 400])
def test_same_results_again_on_another_stream_and_captured(t):
    x, w, a, b, dy = _inputs(t, 1024, 768, 3, 16, torch.bfloat16)
    rows = adapter_rows([0, 3, t - 4, t], [0, 2, 1], device=DEV)
    want = _train(x, w, a, b, rows, 1.0, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _train(x, w, a, b, rows, 1.0, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(again[n], v) for n, v in want.items())
    # two graphs whose replays overlap: nothing is shared but the inputs
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_train(x, w, a, b, rows, 1.0, dy))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for out in outs:
        assert all(torch.equal(out[n], v) for n, v in want.items())


@pytest.mark.parametrize("t", [17, 400])
@pytest.mark.parametrize("slot", [-1, 1])
def test_inputs_made_just_before(t, slot):
    """Every kernel begins while the one before it ends: inputs that the stream has only just filled, by copies, memsets
    and kernels, eagerly and captured, are those that count."""
    x, w, a, b, dy = _inputs(t, 1024, 768, 2, 16, torch.bfloat16)
    rows = adapter_rows([0, t], [slot], device=DEV)
    want = _train(x, w, a, b, rows, 1.0, dy)
    live = [torch.empty_like(v) for v in (x, w, a, b, dy)]
    big = torch.randn(64, 1 << 20, device=DEV)

    def fill_and_run():
        for v in live:
            v.zero_()
        big.mul_(1.0)
        for v, of in zip(live, (x, w, a, b, dy)):
            v.copy_(of)
        out = _train(*live[:4], rows, 1.0, live[4])
        for v in live:               # ... and are read before the stream's next work overwrites them
            v.fill_(math.nan)
        return out

    for _ in range(5):
        got = fill_and_run()
        assert all(torch.equal(got[n], v) for n, v in want.items())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fill_and_run()
    for _ in range(5):
        g.replay()
        assert all(torch.equal(got[n], v) for n, v in want.items())
    w2, a2 = w[:, :768].contiguous(), a[:, :, :768].contiguous()      # a projection of what another one made
    chained = adapter_linear(adapter_linear(x, w, a, b, rows), w2, a2, b, rows)
    torch.cuda.synchronize()
    mid = adapter_linear(x, w, a, b, rows)
    torch.cuda.synchronize()
    assert torch.equal(chained, adapter_linear(mid, w2, a2, b, rows))


def test_gradients_against_differences():
    """A direction's derivative of a weighted sum of y, from y alone."""
    x, w, a, b, dy = _inputs(150, 256, 256, 2, 8, torch.float16)
    cu, slots = [0, 60, 150], [1, 0]
    got = _train(x, w, a, b, adapter_rows(cu, slots, device=DEV), 1.0, dy)
    g = torch.Generator(device=DEV).manual_seed(5)
    for name, v in (("dx", x), ("da", a), ("db", b)):
        way = torch.randn(v.shape, device=DEV, generator=g, dtype=torch.float64)
        sides = []
        for e in (0.5, -0.5):
            moved = {n: t.double() + (e * way if t is v else 0) for n, t in (("x", x), ("a", a), ("b", b))}
            y = moved["x"] @ w.double().t()
            for lo, hi, s in ((0, 60, 1), (60, 150, 0)):
                y[lo:hi] += moved["x"][lo:hi] @ moved["a"][s].t() @ moved["b"][s].t()
            sides.append((y * dy.double()).sum())
        # y is linear in each of its three inputs by itself: the central difference is exact
        _, bound = oracle(x, w, a, b, cu, slots, 1.0, dy)[name]
        assert abs((got[name].double() * way).sum() - (sides[0] - sides[1])) <= (bound * way.abs()).sum() + 1e-6


def test_refusals():
    x, w, a, b, _ = _inputs(16, 64, 64, 2, 8, torch.bfloat16)
    rows = adapter_rows([0, 16], [1], device=DEV)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        adapter_linear(x.float(), w.float(), a.float(), b.float(), rows)
    with pytest.raises(TypeError, match="weight is"):
        adapter_linear(x, w.half(), a, b, rows)
    with pytest.raises(ValueError, match="multiples of 8"):
        adapter_linear(x[:, :60], w[:, :60], a[:, :, :60], b, rows)
    with pytest.raises(ValueError, match="rank 4"):
        adapter_linear(x, w, a[:, :4], b[:, :, :4], rows)
    with pytest.raises(ValueError, match="rank 136"):
        adapter_linear(x, w, a.repeat(1, 17, 1), b.repeat(1, 1, 17), rows)
    with pytest.raises(ValueError, match="cover 16 rows"):
        adapter_linear(x[:8], w, a, b, rows)
    with pytest.raises(ValueError, match="slot 1 of a stack of 1"):
        adapter_linear(x, w, a[:1], b[:1], rows)
    with pytest.raises(TypeError, match="laid out for cpu"):
        adapter_linear(x, w, a, b, adapter_rows([0, 16], [1], device="cpu"))
    with pytest.raises(ValueError, match="freeze"):
        h = [v.half() for v in (x, w, a, b)]
        adapter_linear(h[0], h[1].requires_grad_(), h[2], h[3], rows)
    with pytest.raises(ValueError, match="scale"):
        adapter_linear(x, w, a, b, rows, torch.ones(3, device=DEV))
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(adapter_linear(leaf, w, a, b, rows).float().sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            adapter_linear(torch.autograd.forward_ad.make_dual(x, x), w, a, b, rows)
