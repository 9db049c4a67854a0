"""Adapters beside a shared projection on the CPU: the PyTorch form, the plan of a batch, refusals."""

import pytest
import torch

from adapter_oracle import row_slots
from bridge_b200.ops import adapter_linear, adapter_rows


def _inputs(t, k, n, s, r, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(t, k, generator=g, dtype=dtype), torch.randn(n, k, generator=g, dtype=dtype)
    a, b = torch.randn(s, r, k, generator=g, dtype=dtype), torch.randn(s, n, r, generator=g, dtype=dtype)
    return [v.requires_grad_() for v in (x, w, a, b)]


def test_gradients_against_differences():
    x, w, a, b = _inputs(7, 5, 6, 3, 2)
    rows = adapter_rows([0, 2, 2, 3, 7], [1, 0, -1, 0], device="cpu")
    scale = torch.tensor([2.0, -0.5, 1.0], dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda *v: adapter_linear(*v, rows, scale), (x, w, a, b))
    y = adapter_linear(x, w, a, b, rows, 0.7)
    for t in range(7):
        s = [1, 1, -1, 0, 0, 0, 0][t]
        merged = w + (0.7 * b[s] @ a[s] if s >= 0 else 0)
        assert torch.allclose(y[t], merged @ x[t])
    grads = torch.autograd.grad(y.sum(), (a, b))
    assert grads[0][2].abs().sum() == 0 and grads[1][2].abs().sum() == 0


def test_batch_dimensions_and_no_rows():
    x, w, a, b = _inputs(6, 8, 8, 1, 8)
    rows = adapter_rows([0, 6], [0], device="cpu")
    y = adapter_linear(x.view(2, 3, 8), w, a, b, rows)
    assert torch.equal(y.reshape(6, 8), adapter_linear(x, w, a, b, rows))
    none = adapter_rows([0], [], device="cpu")
    y = adapter_linear(x[:0], w, a, b, none)
    assert y.shape == (0, 8)
    assert all(g.abs().sum() == 0 for g in torch.autograd.grad(y.sum(), (x, w, a, b)))


@pytest.mark.parametrize("seed", range(6))
def test_plan(seed):
    """Every row is named once: by its tile's pairs and by its slot's blocks."""
    g = torch.Generator().manual_seed(seed)
    count = int(torch.randint(1, 60, (), generator=g))
    longest = [3, 40, 900][seed % 3]
    lengths = torch.randint(0, longest, (count,), generator=g).tolist()
    slots = torch.randint(-1, [1, 5, 40][seed // 2], (count,), generator=g).tolist()
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    rows = adapter_rows(cu, slots, device="cpu")
    total, top, units, blocks, o_row, o_tile, o_pair, o_first, o_unit, o_start, o_block = rows.meta
    table = rows.table.tolist()
    want = row_slots(cu, slots, "cpu").tolist()
    assert total == cu[-1] and top == max(slots) + 1 and table[o_row:o_row + total] == want
    assert all(o % 4 == 0 for o in (o_row, o_tile, o_pair, o_first, o_unit, o_start, o_block))
    seen = [-1] * total
    for t in range(-(-total // 256)):
        for p in range(table[o_tile + t], table[o_tile + t + 1]):
            pair = table[o_pair + 12 * p:o_pair + 12 * p + 12]
            for i in range(256):
                if not pair[4 + i // 32] >> (i % 32) & 1:
                    assert seen[256 * t + i] == -1
                    seen[256 * t + i] = pair[0]
    assert seen == want
    seen = [-1] * total
    for u in range(units):
        unit = table[o_unit + 8 * u:o_unit + 8 * u + 8]
        assert table[o_first + unit[0]] <= u < table[o_first + unit[0] + 1]
        here = [i for i in range(128) if not unit[4 + i // 32] >> (i % 32) & 1]
        assert here
        for i in here:
            assert seen[128 * unit[0] + i] == -1
            seen[128 * unit[0] + i] = unit[1]
    assert seen == want
    seen = [-1] * total
    assert table[o_start] == 0 and table[o_start + top] == blocks
    for s in range(top):
        last = -1
        for at in range(table[o_start + s], table[o_start + s + 1]):
            row, n, slot, _ = table[o_block + 4 * at:o_block + 4 * at + 4]
            assert 1 <= n <= 64 and row > last and slot == s
            last = row + n - 1
            assert seen[row:row + n] == [-1] * n
            seen[row:row + n] = [s] * n
    assert seen == want


def test_refusals():
    x, w, a, b = _inputs(4, 8, 8, 2, 8)
    rows = adapter_rows([0, 4], [1], device="cpu")
    for cu, slots in (([0, 4], []), ([1, 4], [0]), ([0, 3, 2], [0, 0]), ([0, 4], [-2])):
        with pytest.raises(ValueError):
            adapter_rows(cu, slots, device="cpu")
    with pytest.raises(ValueError, match="cover 4 rows"):
        adapter_linear(x[:3], w, a, b, rows)
    with pytest.raises(ValueError, match="slot 1 of a stack of 1"):
        adapter_linear(x, w, a[:1], b[:1], rows)
    with pytest.raises(ValueError, match="do not fit"):
        adapter_linear(x, w, a, b[:, :, :4], rows)
    with pytest.raises(ValueError, match="dimensions"):
        adapter_linear(x, w, a[0], b, rows)
    with pytest.raises(TypeError, match="b is"):
        adapter_linear(x, w, a, b.float(), rows)
    with pytest.raises(TypeError, match="adapter_rows"):
        adapter_linear(x, w, a, b, [0, 4])
    with pytest.raises(ValueError, match="scale"):
        adapter_linear(x, w, a, b, rows, torch.ones(3))
