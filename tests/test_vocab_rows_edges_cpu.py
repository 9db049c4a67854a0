"""The PyTorch form of the operators over rows of logits where it can go wrong."""

import math

import pytest
import torch

from bridge_b200.ops import token_logprobs
from tests import vocab_oracle as oracle
from tests.test_vocab_rows_cpu import _case


def test_rows_of_finite_masks_carry_nothing():
    for fill in (-1e10, -1e15, -1e25):
        x = torch.full((2, 30), fill).requires_grad_()
        r = token_logprobs(x, torch.tensor([1, 2]), top_k=3)
        assert r.logp.tolist() == [-math.inf] * 2 and r.entropy.tolist() == [0.0] * 2
        (g,) = torch.autograd.grad((r.logp, r.entropy), x, (torch.ones(2), torch.ones(2)))
        assert not g.any()
    x = torch.zeros(2, 30)
    x[1, 4] = 3e10
    assert torch.isnan(token_logprobs(x, torch.tensor([1, 4])).logp).tolist() == [False, True]
