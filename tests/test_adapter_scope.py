"""What adapters on a whole model leave out, and what the engine does not do with them, is said and not passed over."""

import warnings

import pytest
import torch

from bridge_b200.engine import AdamWConfig, EngineConfig, MixedPrecisionAdamW, TPREngine
from bridge_b200.models import AdapterSet, build_model, get_config
from tests.helpers import flat_ppo_loss, rel_err, set_old_log_probs, tree_batch


def test_experts_without_adapters_are_named():
    model = build_model(get_config("tiny_moe"), seed=1, dtype=torch.float32)
    with pytest.warns(UserWarning, match="experts of . mixture-of-experts layers"):
        AdapterSet(model, slots=1, rank=8)


@pytest.mark.parametrize("preset,targets", [("tiny_moe", ("qkv", "o_proj")), ("tiny", ("qkv", "fc1", "fc2"))])
def test_no_warning_where_nothing_is_left_out(preset, targets):
    model = build_model(get_config(preset), seed=1, dtype=torch.float32)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        AdapterSet(model, slots=1, rank=8, targets=targets)


def _engine(executor="forest", mode="retain"):
    cfg = get_config("tiny")
    return TPREngine(cfg, EngineConfig(executor=executor, forest_mode=mode, token_budget=80), device="cpu",
                     model=build_model(cfg, dtype=torch.float32, seed=0))


def _filled(model):
    adapters = AdapterSet(model, slots=2, rank=8, seed=3)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for p in adapters.b.values():
            p.copy_(torch.randn(p.shape, generator=g) * 0.05)
    return adapters


@pytest.mark.parametrize("executor,mode", [("forest", "retain"), ("forest", "recompute"), ("segment", "retain")])
def test_one_slot_through_the_engine(executor, mode):
    """The engine's schedules against the flattened batch (tolerances: test_models_cpu's, FP32 sums in another order)."""
    batch = tree_batch(n_trees=2, prefix=48, siblings=3, resp=16, seed=7)
    ref = build_model(get_config("tiny"), dtype=torch.float32, seed=0)
    set_old_log_probs(ref, batch)
    plain = _filled(ref)
    with plain.use(1):
        loss, _ = flat_ppo_loss(ref, batch)
        loss.backward()
    eng = _engine(executor, mode)
    adapters = _filled(eng.model)
    with adapters.use(1):
        out = eng.forward_backward_batch(batch)
    assert abs(out["loss"][0] - loss.item()) < 1e-5 * max(1, abs(loss.item()))
    for (name, p), q in zip(adapters.named_parameters(), plain.parameters()):
        assert (p.grad[0] == 0).all() and rel_err(p.grad[1], q.grad[1]) < 2e-4, name


def test_the_engine_does_not_step_a_model_with_adapters():
    eng = _engine()
    batch = tree_batch(n_trees=1, prefix=8, siblings=2, resp=4, seed=7)
    set_old_log_probs(eng.model, batch)
    adapters = _filled(eng.model)
    before = [p.detach().clone() for p in eng.model.parameters()]
    with adapters.use(0):
        for step in (lambda: eng.train_step(batch), eng.optimizer_step):
            with pytest.raises(NotImplementedError, match="AdapterSet"):
                step()
    assert all(torch.equal(p, q) for p, q in zip(eng.model.parameters(), before))
    with pytest.raises(ValueError, match="takes a gradient"):
        TPREngine(get_config("tiny"), EngineConfig(), device="cpu", model=eng.model)
    adapters.remove()
    eng.model.requires_grad_(True)
    eng.train_step(batch)
    assert any(not torch.equal(p, q) for p, q in zip(eng.model.parameters(), before))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["retain", "recompute"])
def test_one_slot_through_the_engine_on_gpu(mode):
    """As above in BF16, into the FP32 accumulators of an optimizer over the adapters: some 40 roundings (half a step: 2^-8)
    of activations, low-rank values and gradients on the way through three layers, in other places: sqrt(40) 2^-8 = 2.5% of
    a gradient's length, allowed three times."""
    cfg = get_config("tiny", hidden_size=512, num_heads=8, num_kv_heads=2, head_dim=128, intermediate_size=1024,
                     num_layers=3)
    batch = tree_batch(n_trees=2, prefix=200, siblings=4, resp=96, seed=5)
    ref = build_model(cfg, device="cuda", seed=0)
    set_old_log_probs(ref, batch)
    plain = _filled(ref)
    with plain.use(1):
        loss, _ = flat_ppo_loss(ref, batch)
        loss.backward()
    eng = TPREngine(cfg, EngineConfig(forest_mode=mode, token_budget=1024), device="cuda",
                    model=build_model(cfg, device="cuda", seed=0))
    adapters = _filled(eng.model)
    optimizer = MixedPrecisionAdamW(adapters, AdamWConfig(grad_clip=0.0))
    with adapters.use(1):
        out = eng.forward_backward_batch(batch)
    assert abs(out["loss"][0] - loss.item()) <= 2e-3 * abs(loss.item()) + 1e-4
    for (name, p), q in zip(adapters.named_parameters(), plain.parameters()):
        got, want = p.main_grad[1], q.grad[1].float()
        assert (p.main_grad[0] == 0).all() and (got - want).norm() <= 0.075 * want.norm(), name
    before = [p.detach().clone() for p in adapters.parameters()]
    adapters.clip_grad_norm_(1.0)
    optimizer.step()
    assert all(torch.isfinite(p).all() for p in adapters.parameters())
    assert any(not torch.equal(p[1], q[1]) for p, q in zip(adapters.parameters(), before))
