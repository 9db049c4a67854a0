"""Measured cases of the vocabulary operators: token log-probs with alternatives, and distillation.

Two operators over rows of logits ``x [U, V]`` (``V`` the vocabulary, ``T`` a temperature per row):

* ``token_logprobs``: ``logp[u, j] = z[u, t_uj] - lse(z[u])`` of given tokens (``z = x / T``), the
  entropy of the row, and its ``k`` likeliest tokens (ties to the lower id); as a training step also
  the gradient of both outputs with respect to ``x``.
* ``topk_distill_loss``: ``KL(q || p)`` of a teacher that is known by its top log-probs only, either
  with one more class for everything outside them (``tail``) or with the given ones renormalised;
  the loss is ``sum_u w_u KL_u / denom``, and a training step also returns ``dloss / dx``.

``run`` computes them from elementary torch operations in 32 bits, or, where ``own`` is true, by the
framework's own calls.  ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_VOCAB = 151936          # vocabulary of the framework's full-size model presets
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # alternatives of ONE decoded position: a call's latency
        dict(name="score_one", op="score", rows=1, vocab=_VOCAB, pad=293, dtype="bf16", tokens=1, top=20,
             entropy=True, temp=1.0, train=False),
        # a short answer scored with a handful of alternatives
        dict(name="score_answer", op="score", rows=37, vocab=_VOCAB, pad=293, dtype="bf16", tokens=1, top=5,
             entropy=True, temp=0.7, train=False),
        # one LM-head chunk of a policy update: log-probs of the taken tokens and the entropy metric
        dict(name="score_chunk", op="score", rows=4096, vocab=_VOCAB, pad=0, dtype="bf16", tokens=1, top=0,
             entropy=True, temp=1.0, train=False),
        # a teacher's pass: only its top log-probs are wanted
        dict(name="teacher_top64", op="score", rows=1024, vocab=_VOCAB, pad=293, dtype="bf16", tokens=0, top=64,
             entropy=False, temp=1.0, train=False),
        # FP32 logits of a small odd vocabulary
        dict(name="score_f32_odd", op="score", rows=515, vocab=5003, pad=0, dtype="f32", tokens=1, top=8,
             entropy=True, temp=1.3, train=False),
        # policy gradient with an entropy bonus: both directions
        dict(name="score_train", op="score", rows=2048, vocab=_VOCAB, pad=0, dtype="bf16", tokens=1, top=0,
             entropy=True, temp=1.0, train=True),
        # several candidate tokens per position (listwise scoring), FP16, both directions
        dict(name="score_train_f16", op="score", rows=300, vocab=5000, pad=0, dtype="f16", tokens=8, top=0,
             entropy=True, temp=0.7, train=True),
        # distillation of a few rows: latency
        dict(name="distill_few", op="distill", rows=8, vocab=_VOCAB, pad=0, dtype="bf16", top=20, tail=True,
             temp=1.0, train=True),
        # one LM-head chunk of a distillation update
        dict(name="distill_chunk", op="distill", rows=4096, vocab=_VOCAB, pad=0, dtype="bf16", top=64, tail=True,
             temp=1.0, train=True),
        # FP32 logits, many teacher entries, renormalised, odd vocabulary
        dict(name="distill_f32_renorm", op="distill", rows=1024, vocab=32003, pad=0, dtype="f32", top=128,
             tail=False, temp=2.0, train=True),
        # held-out loss only
        dict(name="distill_eval", op="distill", rows=1024, vocab=_VOCAB, pad=293, dtype="bf16", top=64, tail=True,
             temp=1.0, train=False),
        # a tiny test-sized model in FP16, with a loss scale
        dict(name="distill_f16_tiny", op="distill", rows=64, vocab=1024, pad=0, dtype="f16", top=8, tail=True,
             temp=1.0, train=True),
    ]


def draw(rng):
    """A case of the same ranges; at most the logits of the largest listed case."""
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = rng.choice([_VOCAB, _VOCAB // 2, _VOCAB // 4, spread(1024, _VOCAB), spread(1024, _VOCAB) | 1])
    width = 4 if dtype == "f32" else 2
    rows = min(spread(1, 4096), (4096 * _VOCAB * 2) // (vocab * width))
    pad = rng.choice([0, 0, vocab // 500])
    case = dict(rows=rows, vocab=vocab, pad=pad, dtype=dtype, temp=rng.choice([1.0, 1.0, 0.7, 1.3]),
                train=rng.random() < 0.5)
    if rng.random() < 0.5:
        case.update(op="score", tokens=rng.choice([1, 1, spread(2, 16)]), entropy=True,
                    top=0 if case["train"] else rng.choice([0, spread(1, 128)]))
    else:
        case.update(op="distill", top=spread(1, 128), tail=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------------------ inputs
def _logits(case, g):
    """Logits as a head gives them: a broad bulk and, in every row, a few dozen tokens that stand out."""
    rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    x = torch.empty(rows, vocab, device="cuda", dtype=dtype)
    likely = torch.randint(0, vocab - case["pad"], (rows, 48), device="cuda", generator=g)
    boost = 4.0 + 5.0 * torch.randn(rows, 48, device="cuda", generator=g).abs()
    for s in range(0, rows, 512):
        part = 2.0 * torch.randn(min(512, rows - s), vocab, device="cuda", generator=g)
        part.scatter_add_(1, likely[s:s + 512], boost[s:s + 512])
        x[s:s + 512] = part
    if case["pad"]:       # columns that only round the vocabulary up carry no token
        x[:, vocab - case["pad"]:] = -math.inf
    return x, likely


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    x, likely = _logits(case, g)
    temp = case["temp"]
    if temp != 1.0:       # one temperature per row, as sampled batches mix them
        temp = temp * (0.8 + 0.4 * torch.rand(rows, device="cuda", generator=g))
    state = {"case": case, "logits": x.requires_grad_(case["train"]), "temp": temp}
    if case["op"] == "score":
        n = case["tokens"]
        if n:
            pick = torch.randint(0, 48, (rows, n), device="cuda", generator=g)
            other = torch.randint(0, vocab - case["pad"], (rows, n), device="cuda", generator=g)
            rare = torch.rand(rows, n, device="cuda", generator=g) < 0.25
            tokens = torch.where(rare, other, likely.gather(1, pick))
            state["tokens"] = tokens[:, 0].contiguous() if n == 1 else tokens
        if case["train"]:
            shape = (rows,) if n == 1 else (rows, n)
            state["d_logp"] = torch.randn(shape, device="cuda", generator=g)
            state["d_entropy"] = 0.1 * torch.randn(rows, device="cuda", generator=g)
        return state
    k = case["top"]
    ids = torch.empty(rows, k, device="cuda", dtype=torch.int64)
    logq = torch.empty(rows, k, device="cuda")
    for s in range(0, rows, 512):     # the teacher: the student's logits, blurred and moved
        part = x.detach()[s:s + 512].float()
        t = 0.8 * part + torch.randn(part.shape, device="cuda", generator=g)
        if torch.is_tensor(temp):
            t = t / temp[s:s + 512, None]
        top = torch.topk(t, k, dim=1)
        ids[s:s + 512] = top.indices
        logq[s:s + 512] = top.values - torch.logsumexp(t, dim=1, keepdim=True)
    if k > 1:                         # a teacher that kept fewer entries in some rows
        kept = torch.randint(max(1, k // 2), 2 * k, (rows, 1), device="cuda", generator=g)
        ids[torch.arange(k, device="cuda")[None] >= kept] = -1
    state.update(ids=ids, logq=logq, weights=0.5 + torch.rand(rows, device="cuda", generator=g), denom=float(rows),
                 scale=16384.0 if case["dtype"] == "f16" and case["train"] else 1.0)
    return state


# ------------------------------------------------------------------------------------- plain forms
def _shifted(state):
    x = state["logits"].detach().float()
    temp = state["temp"]
    top = x.amax(dim=1, keepdim=True)
    return x, (x - top) / (temp[:, None] if torch.is_tensor(temp) else temp)


def _per_row(temp):
    return temp[:, None] if torch.is_tensor(temp) else temp


def _plain_score(state):
    case = state["case"]
    x, d = _shifted(state)
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    log_s = torch.log(s)
    out = {}
    if case["entropy"]:
        d0 = torch.where(e > 0, d, torch.zeros_like(d))
        mean = (e * d0).sum(dim=1, keepdim=True) / s
        out["entropy"] = (log_s - mean)[:, 0]
    if case["tokens"]:
        tokens = state["tokens"].view(case["rows"], -1)
        out["logp"] = (d.gather(1, tokens) - log_s).view(state["tokens"].shape)
    if case["top"]:
        bits = (x + 0.0).view(torch.int32)       # + 0.0: one zero
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        order |= torch.arange(case["vocab"] - 1, -1, -1, device=x.device)
        ids = case["vocab"] - 1 - (torch.topk(order, case["top"], dim=1).values & 0xFFFFFFFF)
        out["top_ids"] = ids
        out["top_logp"] = d.gather(1, ids) - log_s
    if case["train"]:
        p = e / s
        g = state["d_logp"].view(case["rows"], -1)
        grad = -p * g.sum(dim=1, keepdim=True)
        grad.scatter_add_(1, tokens, g)
        grad -= state["d_entropy"][:, None] * p * (d0 - mean)
        out["grad"] = (grad / _per_row(state["temp"])).to(state["logits"].dtype)
    return out


def _plain_distill(state):
    case = state["case"]
    _, d = _shifted(state)
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    logp = d - torch.log(s)
    held = state["ids"] >= 0
    ids = state["ids"].clamp(min=0)
    logq = torch.where(held, state["logq"], torch.full_like(state["logq"], -math.inf))
    if not case["tail"]:
        top = logq.amax(dim=1, keepdim=True)
        logq = logq - (top + torch.log(torch.exp(logq - top).sum(dim=1, keepdim=True)))
    q = torch.exp(logq)
    gap = torch.where(held, logq - logp.gather(1, ids), torch.zeros_like(q))
    rows = (q * gap).sum(dim=1, keepdim=True)
    given = torch.zeros_like(e, dtype=torch.bool).scatter_(1, ids, held)
    # a dropped entry points at token 0: put back what a held entry there says
    given[:, :1] = (held & (ids == 0)).any(dim=1, keepdim=True)
    if case["tail"]:
        q_rest = (1.0 - q.sum(dim=1, keepdim=True)).clamp(min=0.0)
        p_rest = torch.where(given, torch.zeros_like(e), e).sum(dim=1, keepdim=True) / s
        rows = rows + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - torch.log(p_rest)),
                                  torch.zeros_like(q_rest))
    weight = state["weights"][:, None]
    out = {"loss": (rows * weight).sum() / state["denom"], "rows": rows[:, 0]}
    if case["train"]:
        p = e / s
        if case["tail"]:
            grad = torch.where(given, p, p * (1.0 - q_rest / p_rest))
        else:
            grad = p
        grad = grad.scatter_add(1, ids, torch.where(held, -q, torch.zeros_like(q)))
        grad = grad * (weight * (state["scale"] / state["denom"])) / _per_row(state["temp"])
        out["grad"] = grad.to(state["logits"].dtype)
    return out


# ---------------------------------------------------------------------------------- the two forms
def _own_score(state):
    from bridge_b200.ops import token_logprobs

    case = state["case"]
    x = state["logits"]
    r = token_logprobs(x, state.get("tokens"), state["temp"], top_k=case["top"], with_entropy=case["entropy"])
    out = {}
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
    if case["tokens"]:
        out["logp"] = r.logp.detach()
    if case["top"]:
        out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
    if case["train"]:
        (out["grad"],) = torch.autograd.grad((r.logp, r.entropy), x, (state["d_logp"], state["d_entropy"]))
    return out


def _own_distill(state):
    from bridge_b200.ops import topk_distill_loss

    case = state["case"]
    x = state["logits"]
    loss, rows = topk_distill_loss(x, state["ids"], state["logq"], weights=state["weights"], denom=state["denom"],
                                   temperature=state["temp"], tail=case["tail"], grad_scale=state["scale"])
    out = {"loss": loss.detach(), "rows": rows}
    if case["train"]:
        (out["grad"],) = torch.autograd.grad(loss * state["scale"] if state["scale"] != 1.0 else loss, x)
    return out


def run(state):
    if state["case"]["op"] == "score":
        return _own_score(state) if own else _plain_score(state)
    return _own_distill(state) if own else _plain_distill(state)


def work(case):
    rows, vocab, k = case["rows"], case["vocab"], case["top"]
    width = 4 if case["dtype"] == "f32" else 2
    logits = rows * vocab * width
    grad = logits if case["train"] else 0
    per_row = 4 * (case["temp"] != 1.0)
    if case["op"] == "score":
        n = case["tokens"]
        per_row += 12 * n + 4 * case["entropy"] + 12 * k + (4 * n + 4 if case["train"] else 0)
        # a shift, an exponential and a sum per logit; the entropy's product; the gradient's product
        flops = (3 + 2 * case["entropy"] + 3 * case["train"]) * rows * vocab
    else:
        per_row += 12 * k + 4 + 4
        flops = (3 + 2 * case["train"]) * rows * vocab
    return {"bytes": logits + grad + rows * per_row, "flops": flops}


# ----------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    state = prepare(case, seed)
    parts = [_exact_rows(case, state, slice(a, min(a + 256, case["rows"]))) for a in range(0, case["rows"], 256)]
    out = {name: None if parts[0][name] is None else torch.cat([p[name] for p in parts]) for name in parts[0]}
    if case["op"] == "distill":
        loss = (out["rows"] * state["weights"].double()).sum() / state["denom"]
        out = {"loss": loss, **out}
    return out


def _exact_rows(case, state, at):
    x = state["logits"].detach()[at].double()
    rows = x.shape[0]
    temp = state["temp"][at].double()[:, None] if torch.is_tensor(state["temp"]) else float(state["temp"])
    logp = torch.log_softmax(x / temp, dim=1)
    p = torch.exp(logp)
    out = {}
    if case["op"] == "score":
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        entropy = -plogp.sum(dim=1)
        if case["entropy"]:
            out["entropy"] = entropy
        if case["tokens"]:
            t = state["tokens"][at].reshape(rows, -1)
            out["logp"] = logp.gather(1, t).reshape(state["tokens"][at].shape)
        if case["top"]:
            out["top_ids"] = None
            out["top_logp"] = torch.topk(logp, case["top"], dim=1).values
        if case["train"]:
            up = state["d_logp"][at].double().reshape(rows, -1)
            grad = torch.zeros_like(p).scatter_add_(1, t, up) - p * up.sum(dim=1, keepdim=True)
            # d entropy / d z_v = -p_v (log p_v + entropy)
            grad -= state["d_entropy"][at].double()[:, None] * (plogp + p * entropy[:, None])
            out["grad"] = grad / temp
        return out
    # one more column takes the entries that were dropped
    ids = torch.where(state["ids"][at] < 0, torch.full_like(state["ids"][at], case["vocab"]), state["ids"][at])
    q = torch.zeros(rows, case["vocab"] + 1, dtype=torch.float64, device=x.device)
    q = q.scatter_(1, ids, torch.exp(state["logq"][at].double()))[:, :-1]
    given = torch.zeros(rows, case["vocab"] + 1, dtype=torch.bool, device=x.device).scatter_(1, ids, True)[:, :-1]
    if not case["tail"]:
        q = q / q.sum(dim=1, keepdim=True)
    kl = torch.where(q > 0, q * (torch.log(q) - logp), torch.zeros_like(q)).sum(dim=1)
    target = q
    if case["tail"]:
        left = (1.0 - q.sum(dim=1)).clamp(min=0.0)
        rest = torch.where(given, torch.zeros_like(p), p).sum(dim=1)
        kl = kl + torch.where(left > 0, left * (torch.log(left) - torch.log(rest)), torch.zeros_like(left))
        # outside the given tokens the target follows the student's own proportions
        target = torch.where(given, q, p * (left / rest)[:, None])
    out["rows"] = kl
    if case["train"]:
        total = target.sum(dim=1, keepdim=True)
        scale = state["weights"][at].double()[:, None] * (state["scale"] / state["denom"])
        out["grad"] = (p * total - target) * scale / temp
    return out
