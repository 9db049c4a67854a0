"""Definitions in 64 bits of the operators over rows of logits (log-probs with alternatives, distillation)."""

from __future__ import annotations

import math

import torch

LOWEST = -6.9e29      # a scaled logit below this is a mask


def scaled(x, temp):
    t = temp.double()[:, None] if torch.is_tensor(temp) else float(temp)
    z = x.double() / t
    return torch.where(z < LOWEST, torch.full_like(z, -math.inf), z)


def log_softmax(z):
    m = z.amax(dim=1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    return z - m - torch.log(torch.exp(z - m).sum(dim=1, keepdim=True))


def token_logprobs(x, tokens, temp, total=None):
    """``(logp [U, n], entropy [U])``; rows without a live logit: -inf and 0."""
    z = scaled(x, temp)
    dead = (z == -math.inf).all(dim=1)
    logp = log_softmax(z)
    p = torch.exp(logp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(dim=1)
    entropy = torch.where(dead, torch.zeros_like(entropy), entropy)
    if tokens is None:
        return None, entropy
    held = (tokens >= 0) & (tokens < (total or x.shape[1]))
    got = logp.gather(1, torch.where(held, tokens, torch.zeros_like(tokens)))
    got = torch.where(dead[:, None], torch.full_like(got, -math.inf), got)
    return torch.where(held, got, torch.zeros_like(got)), entropy


def token_grad(x, tokens, temp, d_logp, d_entropy):
    z = scaled(x, temp)
    dead = (z == -math.inf).all(dim=1, keepdim=True)
    logp = log_softmax(z)
    p = torch.where(dead, torch.zeros_like(z), torch.exp(logp))
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    g = torch.zeros_like(p)
    if tokens is not None and d_logp is not None:
        held = (tokens >= 0) & (tokens < x.shape[1]) & ~dead
        d = torch.where(held, d_logp.double(), torch.zeros_like(d_logp.double()))
        g.scatter_add_(1, torch.where(held, tokens, torch.zeros_like(tokens)), d)
        g = g - p * d.sum(dim=1, keepdim=True)
    if d_entropy is not None:
        g = g - d_entropy.double()[:, None] * (plogp - p * plogp.sum(dim=1, keepdim=True))
    t = temp.double()[:, None] if torch.is_tensor(temp) else float(temp)
    return g / t


def top(x, k):
    """Ids of the k largest, ties to the lower id (NaN as -inf)."""
    v = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).double()
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]


def distill(x, ids, logq, temp, tail):
    """``(KL [U], dKL/dx [U, V])`` with entries kept one by one (repeats included)."""
    vocab = x.shape[1]
    logp_all = log_softmax(scaled(x, temp))
    kl, grad = [], []
    t = temp.double() if torch.is_tensor(temp) else torch.full((x.shape[0],), float(temp), dtype=torch.float64,
                                                               device=x.device)
    for u in range(x.shape[0]):
        logp = logp_all[u]
        keep = (ids[u] >= 0) & (ids[u] < vocab)
        i, lq = ids[u][keep], logq[u][keep].double()
        if not tail and i.numel():
            lq = lq - torch.logsumexp(lq, 0)
        if i.numel() == 0 or (not tail and bool(torch.isnan(lq).any())):
            kl.append(logp.new_zeros(()))
            grad.append(torch.zeros_like(logp))
            continue
        q = torch.exp(lq)
        value = torch.where(q == 0, torch.zeros_like(q), q * (lq - logp[i])).sum()
        target = torch.zeros_like(logp).index_add_(0, i, q)
        p = torch.exp(logp)
        total = q.sum()
        if tail:
            given = torch.zeros_like(logp, dtype=torch.bool)
            given[i] = True
            left = (1.0 - q.sum()).clamp(min=0.0)
            rest = p[~given].sum()
            if left > 0:
                value = value + left * (torch.log(left) - torch.log(rest))
                total = total + left
                if rest > 0:
                    target = target + torch.where(given, torch.zeros_like(p), p * (left / rest))
        kl.append(value)
        grad.append((p * total - target) / t[u])
    return torch.stack(kl), torch.stack(grad)
