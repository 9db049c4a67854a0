"""Adapters on whole models, with the clipping and the optimizer that follow: a run of them as it would be used."""

import gc
import weakref

import pytest
import torch

from bridge_b200.engine.optim import AdamWConfig, MixedPrecisionAdamW
from bridge_b200.models import AdapterSet, build_model, get_config
from bridge_b200.ops import adapter_rows

LENGTHS, SLOTS = [40, 24, 33, 7], [1, -1, 0, 1]


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _filled(model, slots=2, rank=8):
    adapters = AdapterSet(model, slots=slots, rank=rank, alpha=2.0 * rank, seed=3)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for p in adapters.b.values():
            p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    return adapters


@pytest.mark.parametrize("preset", ["tiny", "tiny_hybrid", "tiny_moe"])
def test_each_projection_is_a_merged_one_on_cpu(preset):
    """Every adapted projection against its weight plus the slot's product, in 64 bits (FP32 sums of K and R products,
    a step of 2^-24 each at most)."""
    cfg = get_config(preset)
    model = build_model(cfg, seed=1, dtype=torch.float32)
    ids = torch.randint(0, cfg.vocab_size, (37,), generator=torch.Generator().manual_seed(0))
    pos = torch.arange(37)
    before = model(ids, pos, 37)
    adapters = _filled(model)
    assert not any(p.requires_grad for p in model.parameters())
    assert torch.equal(model(ids, pos, 37), before)
    modules = {name.replace(".", "/"): m for name, m in model.named_modules()}
    g = torch.Generator().manual_seed(2)
    for slot in (-1, 0, 1):
        with adapters.use(slot):
            assert torch.equal(model(ids, pos, 37), before) == (slot < 0)
            for key, a in adapters.a.items():
                m = modules[key]
                x = torch.randn(5, a.shape[2], generator=g)
                a, b = a[slot].detach().double(), adapters.b[key][slot].detach().double()
                c = adapters.scale if slot >= 0 else 0.0
                want = x.double() @ (m.weight.detach().double() + c * b @ a).t()
                size = x.double().abs() @ (m.weight.detach().double().abs() + c * b.abs() @ a.abs()).t()
                assert ((m(x).double() - want).abs() <= (a.shape[1] + a.shape[0] + 4) * 2.0 ** -24 * size).all(), key
    adapters.remove()
    assert all(m.adapter is None for m in model.modules() if hasattr(m, "adapter"))


def _train(device, dtype=None):
    """Two steps of two policies whose requests share the batch's projections; MLP projections are per row, so each
    request's rows can be checked alone."""
    cfg = get_config("tiny")
    model = build_model(cfg, seed=1, dtype=dtype, device=device)
    adapters = _filled(model)
    optimizer = MixedPrecisionAdamW(adapters, AdamWConfig(lr=1e-3, grad_clip=0.0))
    cu = _cu(LENGTHS)
    rows = adapter_rows(cu, SLOTS, device=device)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, cfg.vocab_size, (cu[-1],), generator=g).to(device)
    pos = torch.arange(cu[-1], device=device)
    way = torch.randn(cu[-1], cfg.hidden_size, generator=g).to(device)
    records = []
    for _ in range(2):
        with adapters.use(rows):
            hidden = model(ids, pos, cu[-1])
        # (a linear functional: the mean square of what the last RMSNorm gives is 1 whatever the adapters are, so its
        # gradient would be nothing but rounding)
        (hidden.float() * way).mean().backward()
        raw = [x.clone() for x in adapters.gradients()]
        norms = adapters.clip_grad_norm_(1e-4)
        records.append((raw, norms, [x.clone() for x in adapters.gradients()]))
        optimizer.step()
        optimizer.zero_grad()
    assert all(p.grad is None for p in model.parameters())
    return adapters, records


def _check(adapters, records):
    for raw, norms, clipped in records:
        assert len(raw) == 2 * len(adapters.a) and all(torch.isfinite(x).all() for x in raw)
        for s in range(2):
            norm = torch.stack([x[s].double().square().sum() for x in raw]).sum().sqrt()
            assert norm > 0 and abs(norms[s].double() - norm) <= 1e-6 * norm
            factor = min(1.0, 1e-4 / (float(norm) + 1e-6))
            for x, c in zip(raw, clipped):
                assert torch.allclose(c[s], x[s] * factor, rtol=1e-6, atol=0)


def test_training_run_on_cpu():
    _check(*_train("cpu", torch.float32))


@pytest.mark.gpu
def test_training_run_on_gpu(monkeypatch):
    adapters, records = _train("cuda")
    _check(adapters, records)
    monkeypatch.setenv("BRIDGE_B200_IMPL", "reference")
    _, plain = _train("cuda")
    # some 20 BF16 roundings (half a step: 2^-8) of activations and their gradients on the way through two layers, in
    # other places: sqrt(20) 2^-8 = 1.7 % of a vector's length, allowed three times
    for got, want in zip(records[0][0], plain[0][0]):
        assert (got - want).norm() <= 0.05 * want.norm() + 1e-8


@pytest.mark.gpu
@pytest.mark.parametrize("preset", ["tiny", "tiny_hybrid", "tiny_moe"])
def test_one_slot_on_gpu(preset):
    cfg = get_config(preset)
    model = build_model(cfg, seed=1, device="cuda")
    ids = torch.randint(0, cfg.vocab_size, (130,), device="cuda")
    pos = torch.arange(130, device="cuda")
    base = model(ids, pos, 130)
    adapters = _filled(model)
    assert torch.equal(model(ids, pos, 130), base)
    with torch.no_grad():
        with adapters.use(1):
            got = model(ids, pos, 130).float()
        with adapters.use(adapter_rows([0, 50, 130], [1, 1])):
            assert torch.equal(model(ids, pos, 130).float(), got)
    assert torch.isfinite(got).all() and (got - base.float()).norm() > 0.01 * base.float().norm()


@pytest.mark.gpu
def test_captured_plan_outlives_the_list():
    """A graph reads the plan of its slot again after hundreds of other lengths have come by."""
    model = build_model(get_config("tiny"), seed=1, device="cuda")
    adapters = _filled(model)
    p = next(m for m in adapters._modules_of)
    x = torch.randn(40, p.weight.shape[1], device="cuda", dtype=p.weight.dtype)
    with torch.no_grad(), adapters.use(1):
        want = p.adapter(x, p.weight)
        plan = weakref.ref(adapters.rows_for(x))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = p.adapter(x, p.weight)
        for t in range(41, 641):
            adapters.rows_for(x.expand(t, 40, -1)[:, 0])
        gc.collect()
        assert plan() is not None and adapters.rows_for(x) is plan()
        assert len(adapters._plans) <= 256
        g.replay()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_refusals_on_gpu():
    model = build_model(get_config("tiny"), seed=1, device="cuda")
    for rank in (4, 12, 136):
        with pytest.raises(ValueError, match="multiple of 8"):
            AdapterSet(model, slots=1, rank=rank)
    adapters = AdapterSet(model, slots=1, rank=8)
    g = torch.cuda.CUDAGraph()
    x = torch.zeros(8, 256, device="cuda", dtype=torch.bfloat16)
    adapters.active = 0
    plan = adapters.rows_for(x)                 # made before: the capture takes it
    with torch.cuda.graph(g):
        assert adapters.rows_for(x) is plan
        with pytest.raises(RuntimeError, match="captured"):
            adapter_rows([0, 8], [0], device="cuda")
        x.add_(1.0)
    g.replay()
    assert (x == 1).all()


def test_refusals():
    model = build_model(get_config("tiny"), seed=1)
    with pytest.raises(ValueError, match="slot"):
        AdapterSet(model, slots=0, rank=8)
    with pytest.raises(ValueError, match="no projection"):
        AdapterSet(model, slots=1, rank=8, targets=("gate",))
    adapters = AdapterSet(model, slots=2, rank=8, targets=("qkv",))
    assert len(adapters.a) == model.config.num_layers
    with pytest.raises(ValueError, match="already"):
        AdapterSet(model, slots=1, rank=8)
    with pytest.raises(ValueError, match="slot 2 of 2"):
        with adapters.use(2):
            pass
    with pytest.raises(TypeError, match="adapter_rows"):
        with adapters.use([0, 1]):
            pass
    with pytest.raises(ValueError, match="no gradients"):
        adapters.clip_grad_norm_(1.0)
    with pytest.raises(ValueError, match="rows"):
        with adapters.use(adapter_rows([0, 3], [0], device="cpu")):
            model(torch.zeros(5, dtype=torch.long), torch.arange(5), 5)
