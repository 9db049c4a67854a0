"""Operators over rows of logits on the CPU: the PyTorch form against 64-bit definitions and differences, and
vocabularies in shards over gloo ranks."""

import math

import pytest
import torch

from bridge_b200.ops import (fused_lm_head_token_logprobs, fused_lm_head_topk_distill, token_logprobs,
                             topk_distill_loss)
from tests import vocab_oracle as oracle
from tests.dist_utils import run_ranks


def _case(rows=6, vocab=90, k=7, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    x = (3.0 * torch.randn(rows, vocab, generator=g)).to(dtype)
    x[1, 10:60] = -math.inf
    tokens = torch.randint(0, vocab, (rows, 3), generator=g)
    tokens[2, 1], tokens[3, 2] = tokens[2, 0], -1
    tokens[1] = torch.tensor([1, 70, 3])
    temp = 0.6 + torch.rand(rows, generator=g)
    t = torch.randn(rows, vocab, generator=g)
    t[1, 10:60] = -40.0
    top = torch.topk(t, k, dim=1)
    ids, logq = top.indices.clone(), top.values - torch.logsumexp(t, 1, keepdim=True)
    ids[0, 4:] = -1
    ids[4] = -1
    ids[5, 2] = ids[5, 6]
    w = 0.2 + torch.rand(rows, generator=g)
    return x, tokens, temp, ids, logq, w


def test_token_logprobs_reference():
    x, tokens, temp, *_ = _case()
    x.requires_grad_()
    r = token_logprobs(x, tokens, temp, top_k=9)
    lp, ent = oracle.token_logprobs(x.detach(), tokens, temp)
    assert torch.allclose(r.logp, lp, rtol=1e-6, atol=1e-6) and torch.allclose(r.entropy, ent, rtol=1e-6, atol=1e-6)
    assert torch.equal(r.top_ids, oracle.top(x.detach(), 9))
    d, dh = torch.randn(6, 3).double(), torch.randn(6).double()
    (g,) = torch.autograd.grad((r.logp, r.entropy), x, (d, dh))
    assert torch.allclose(g, oracle.token_grad(x.detach(), tokens, temp, d, dh), rtol=1e-5, atol=1e-6)
    one = token_logprobs(x, tokens[:, 0], 0.9)
    assert one.logp.shape == (6,) and one.top_ids is None


def test_reference_gradients_against_differences():
    _, tokens, _, _, logq, w = _case()
    x = torch.randn(3, 30, dtype=torch.float64).requires_grad_()
    tokens, ids, logq = tokens[:3] % 30, torch.stack([torch.randperm(30)[:4] for _ in range(3)]), logq[:3, :4] - 0.2

    def scores(v):
        r = token_logprobs(v, tokens, 0.8)
        return r.logp, r.entropy

    assert torch.autograd.gradcheck(scores, (x,), eps=1e-5, atol=1e-5)
    for tail in (True, False):
        way = torch.randn(3, 30, dtype=torch.float64)
        loss, _ = topk_distill_loss(x, ids, logq, denom=2.0, weights=w[:3], temperature=0.7, tail=tail)
        (g,) = torch.autograd.grad(loss, x)
        with torch.no_grad():
            up, down = (topk_distill_loss(x + s * 1e-4 * way, ids, logq, denom=2.0, weights=w[:3], temperature=0.7,
                                          tail=tail)[0] for s in (1, -1))
        assert abs(float((g * way).sum()) - float(up - down) / 2e-4) < 1e-5


@pytest.mark.parametrize("tail", [True, False])
def test_distill_reference(tail):
    x, _, temp, ids, logq, w = _case()
    x.requires_grad_()
    loss, rows = topk_distill_loss(x, ids, logq, denom=5.0, weights=w, temperature=temp, tail=tail, grad_scale=2.0)
    kl, g = oracle.distill(x.detach(), ids, logq, temp, tail)
    assert torch.allclose(rows, kl, rtol=1e-6, atol=1e-6)
    assert torch.allclose(loss, (kl * w).sum() / 5.0, rtol=1e-6, atol=1e-6)
    (got,) = torch.autograd.grad(loss * 2.0, x)
    assert torch.allclose(got, g * w.double()[:, None] * 2.0 / 5.0, rtol=1e-5, atol=1e-6)


def test_heads_and_masked_rows():
    g = torch.Generator().manual_seed(1)
    h, W = torch.randn(9, 16, generator=g), torch.randn(40, 16, generator=g)
    t = fused_lm_head_token_logprobs(h, W, None, 1.3, top_k=5, chunk_rows=4)
    assert torch.equal(t.top_ids, oracle.top(h @ W.t(), 5)) and t.logp is None
    hs = (h + 0.1).requires_grad_()
    loss, rows = fused_lm_head_topk_distill(hs, W, t.top_ids, t.top_logp, denom=9.0)
    loss.backward()
    _, gx = oracle.distill(hs.detach() @ W.t(), t.top_ids, t.top_logp, 1.0, True)
    assert torch.allclose(hs.grad.double(), gx @ W.double() / 9.0, rtol=1e-4, atol=1e-5)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        x = torch.full((2, 8), low).requires_grad_()
        r = token_logprobs(x, torch.tensor([1, 2]), top_k=3)
        assert r.logp.tolist() == [-math.inf] * 2 and r.entropy.tolist() == [0.0] * 2
        (gr,) = torch.autograd.grad((r.logp, r.entropy), x, (torch.ones(2), torch.ones(2)))
        assert not gr.any() and r.top_ids.tolist() == [[0, 1, 2]] * 2


def test_refusals_on_cpu():
    x, tokens, *_ , ids, logq, _ = _case()
    for bad in (dict(temperature=0), dict(top_k=91), dict(tokens=tokens[:2])):
        with pytest.raises(ValueError):
            token_logprobs(x, **bad)
    with pytest.raises(TypeError):
        token_logprobs(x.long())
    with pytest.raises(ValueError):
        topk_distill_loss(x, ids, logq, denom=-1.0)


def _shard_worker(rank, world):
    import torch.distributed as dist

    x, tokens, temp, ids, logq, w = _case()
    part = x.shape[1] // world
    mine = x[:, rank * part:(rank + 1) * part].clone().requires_grad_()
    group = dist.group.WORLD
    at = dict(vocab_start=rank * part, tp_group=group)
    r = token_logprobs(mine, tokens, temp, top_k=40, **at)
    d, dh = torch.arange(18.0).view(6, 3).double() / 9 - 1, torch.linspace(-1, 1, 6).double()
    (g1,) = torch.autograd.grad((r.logp, r.entropy), mine, (d, dh))
    out = [r.logp.detach(), r.entropy.detach(), r.top_ids, r.top_logp, g1]
    for tail in (True, False):
        loss, rows = topk_distill_loss(mine, ids, logq, denom=3.0, weights=w, temperature=temp, tail=tail, **at)
        (g,) = torch.autograd.grad(loss, mine)
        out += [loss.detach(), rows, g]
    return [o.tolist() for o in out]


@pytest.mark.parametrize("world", [2, 3])
def test_vocabulary_shards_match_whole_rows(world):
    """Every rank gets the whole result; the shards' gradients side by side are the whole gradient."""
    ranks = [[torch.tensor(v) for v in r] for r in run_ranks(world, _shard_worker)]
    x, tokens, temp, ids, logq, w = _case()
    lp, ent = oracle.token_logprobs(x, tokens, temp)
    d, dh = torch.arange(18.0).view(6, 3).double() / 9 - 1, torch.linspace(-1, 1, 6).double()
    for r in ranks:
        assert torch.allclose(r[0].double(), lp, atol=1e-5) and torch.allclose(r[1].double(), ent, atol=1e-5)
        assert torch.equal(r[2], oracle.top(x, 40))
        assert torch.allclose(r[3].double(), oracle.token_logprobs(x, oracle.top(x, 40), temp)[0], atol=1e-5)
    side = torch.cat([r[4] for r in ranks], 1).double()
    assert torch.allclose(side, oracle.token_grad(x, tokens, temp, d, dh), atol=1e-5)
    for i, tail in ((5, True), (8, False)):
        kl, g = oracle.distill(x, ids, logq, temp, tail)
        for r in ranks:
            assert torch.allclose(r[i].double(), (kl * w).sum() / 3.0, atol=1e-5)
            assert torch.allclose(r[i + 1].double(), kl, atol=1e-5)
        side = torch.cat([r[i + 2] for r in ranks], 1).double()
        assert torch.allclose(side, g * w.double()[:, None] / 3.0, atol=1e-5)
