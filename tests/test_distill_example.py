"""The distillation example end to end: teacher alternatives, student loss, optimizer step, scoring."""

import pytest
import torch

from examples.topk_distillation import run


def _check(history):
    losses = [h["loss"] for h in history]
    assert all(torch.isfinite(torch.tensor(list(h.values()))).all() for h in history)
    assert losses[-1] < 0.8 * losses[0], losses
    assert history[-1]["first_choice_logp"] > history[0]["first_choice_logp"]


@pytest.mark.parametrize("tail", [True, False])
def test_distillation_learns_on_cpu(tail):
    _check(run(rows=48, top_k=8, steps=8, device="cpu", tail=tail))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_learns_on_gpu(tail):
    cfg = dict(rows=200, top_k=32, steps=10, device="cuda", tail=tail, temperature=0.9)
    _check(run(**cfg))


@pytest.mark.gpu
def test_first_step_matches_the_reference_form(monkeypatch):
    """Kernels against the PyTorch form of the same step (BF16 models: 2^-7 of the loss and the log-probs)."""
    own = run(rows=96, top_k=20, steps=1, device="cuda")[0]
    monkeypatch.setenv("BRIDGE_B200_IMPL", "reference")
    ref = run(rows=96, top_k=20, steps=1, device="cuda")[0]
    for k in own:
        assert abs(own[k] - ref[k]) <= 2.0 ** -7 * max(1.0, abs(ref[k])), (k, own, ref)
