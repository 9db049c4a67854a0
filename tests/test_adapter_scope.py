"""What adapters on a whole model leave out, and what the engine does not do with them, is said and not passed over."""

import warnings

import pytest
import torch

from bridge_b200.models import AdapterSet, build_model, get_config


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
