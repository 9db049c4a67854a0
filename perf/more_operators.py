"""Measured cases of the adapter operators: low-rank adapters beside a shared projection, norms and clipping.

* ``adapter_linear``: rows ``x [T, K]`` of a packed batch of requests through one shared weight ``W [N, K]``
  and, beside it, the low-rank adapter of each row's request: ``y_t = W x_t + scale_s B_s (A_s x_t)`` with
  ``s`` the request's slot in ``A [S, R, K]``, ``B [S, N, R]`` (no adapter where ``s = -1``).  A training
  step returns ``dx``, ``dA`` and ``dB`` too (``W`` is frozen).
* ``clip_grad_norm``: the 2-norm over many gradient tensors, of all of them or, where they are stacked by
  slot, of each slot by itself; and the gradients times ``min(1, max_norm / (norm + 1e-6))``, without
  the loss scale that they carry.

``run`` computes them from elementary torch operations in 32 bits (64 for the long sums of squares), or,
where ``own`` is true, by the framework's own calls.  ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token of one request through a QKV projection: a call's latency
        dict(name="token_one", op="linear", rows=1, requests=1, k=2560, n=6144, slots=8, rank=16, dtype="bf16",
             train=False),
        # one new token for each of 32 requests, through an output projection
        dict(name="tokens_32", op="linear", rows=32, requests=32, k=4096, n=2560, slots=16, rank=16, dtype="bf16",
             train=False),
        # a few tokens of each of some requests, an odd count, through a wide projection, FP16
        dict(name="tokens_61_f16", op="linear", rows=61, requests=23, k=2560, n=19456, slots=8, rank=64, dtype="f16",
             train=False),
        # short ragged prompts that share tiles, through a hybrid layer's input projection
        dict(name="prompts_short", op="linear", rows=517, requests=19, k=2048, n=12352, slots=6, rank=8, dtype="bf16",
             train=False),
        # ordinary prompts, FP16, through an MLP's second projection
        dict(name="prompts_f16", op="linear", rows=2047, requests=5, k=9728, n=2560, slots=4, rank=32, dtype="f16",
             train=False),
        # long prompts through an MLP's first projection: the largest forward
        dict(name="prompts_long", op="linear", rows=8192, requests=12, k=2560, n=19456, slots=8, rank=16,
             dtype="bf16", train=False),
        # a tiny model's training step: latency of both directions
        dict(name="train_tiny", op="linear", rows=203, requests=7, k=256, n=512, slots=3, rank=8, dtype="f16",
             train=True),
        # a training step over ragged responses of four policies
        dict(name="train_qkv", op="linear", rows=4608, requests=9, k=2560, n=6144, slots=4, rank=16, dtype="bf16",
             train=True),
        # the largest training step, wide rank
        dict(name="train_wide", op="linear", rows=8192, requests=16, k=9728, n=2560, slots=2, rank=64, dtype="bf16",
             train=True),
        # gradients of a tiny model's adapters: latency
        dict(name="clip_tiny", op="clip", layers=2, hidden=256, ffn=512, slots=1, rank=8, full=False, dtype="f32",
             out="f32", per_slot=False, bound=0.5, scale=1.0),
        # gradients of eight policies' adapters of a full-size model, each policy clipped by its own norm
        dict(name="clip_policies", op="clip", layers=36, hidden=2560, ffn=9728, slots=8, rank=16, full=False,
             dtype="f32", out="f32", per_slot=True, bound=1.0, scale=1.0),
        # all weights' BF16 gradients of a model, with a loss scale, into the FP32 buffers of the optimizer
        dict(name="clip_model", op="clip", layers=12, hidden=2048, ffn=5632, slots=1, rank=0, full=True,
             dtype="bf16", out="f32", per_slot=False, bound=0.5, scale=1024.0),
    ]


def draw(rng):
    """A case of the same ranges; no more products than the largest listed ones, no more gradient bytes."""
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    if rng.random() < 0.3:
        full = rng.random() < 0.3
        case = dict(op="clip", layers=spread(1, 36), hidden=64 * spread(4, 40), ffn=64 * spread(8, 152),
                    slots=1 if full else spread(1, 16), rank=0 if full else 8 * spread(1, 8), full=full,
                    dtype=rng.choice(["f32", "bf16", "f16"]), bound=rng.choice([0.5, 1.0, 3.0]))
        case["out"] = rng.choice(["f32", case["dtype"]])
        case["per_slot"] = not full and rng.random() < 0.6
        case["scale"] = rng.choice([1.0, 1024.0])
        while sum(math.prod(s) for s in _shapes(case)) > 230_000_000:
            case["layers"] = (case["layers"] + 1) // 2
            case["slots"] = (case["slots"] + 1) // 2
            case["hidden"] = max(64, case["hidden"] // 128 * 64)
        return case
    train = rng.random() < 0.5
    k = rng.choice([256, 2048, 2560, 4096, 8 * spread(16, 1216)])
    n = rng.choice([512, 2560, 6144, 12352, 8 * spread(16, 2432)])
    rows = rng.choice([spread(1, 64), spread(1, 8192)])
    rows = max(1, min(rows, 8192 * 2560 * 19456 // (k * n * (2 if train else 1))))
    return dict(op="linear", rows=rows, requests=rows if rows <= 64 and rng.random() < 0.5 else spread(1, min(rows, 48)),
                k=k, n=n, slots=spread(1, 16), rank=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                dtype=rng.choice(["bf16", "bf16", "f16"]), train=train)


# ------------------------------------------------------------------------------------------ inputs
def _requests(case, seed):
    """Where each request begins, and the slot of its adapter; about one in twelve has none."""
    rng = random.Random(seed * 7 + 1)
    cuts = sorted(rng.sample(range(1, case["rows"]), case["requests"] - 1)) if case["requests"] > 1 else []
    cu = [0] + cuts + [case["rows"]]
    slots = [rng.randrange(case["slots"]) for _ in range(case["requests"])]
    return cu, [-1 if i and rng.random() < 1 / 12 else s for i, s in enumerate(slots)]


def _prepare_linear(case, seed, g):
    t, k, n, s, r = (case[i] for i in ("rows", "k", "n", "slots", "rank"))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).to(dtype)

    cu, slots = _requests(case, seed)
    state = {"case": case, "x": normal(t, k), "weight": normal(n, k, std=k ** -0.5),
             "a": normal(s, r, k, std=k ** -0.5), "b": normal(s, n, r, std=0.5 * r ** -0.5), "scale": 2.0,
             "cu": cu, "slots": slots}
    if case["train"]:
        state["dy"] = normal(t, n)
        for name in ("x", "a", "b"):
            state[name].requires_grad_()
    # the rows of each slot, and the framework's plan of the batch: what a program has from its scheduler
    rows = {}
    for i, slot in enumerate(slots):
        if slot >= 0:
            rows.setdefault(slot, []).extend(range(cu[i], cu[i + 1]))
    if own:
        from bridge_b200.ops import adapter_rows

        state["rows"] = adapter_rows(cu, slots, device="cuda")
    else:
        state["rows"] = {slot: torch.tensor(at, device="cuda") for slot, at in rows.items()}
    return state


def _shapes(case):
    h, f, s, r = case["hidden"], case["ffn"], case["slots"], case["rank"]
    weights = [(2 * h, h), (h, h), (2 * f, h), (h, f)]
    layer = []
    for n, k in weights:
        layer += [(n, k)] if case["full"] else [(s, r, k), (s, n, r)]
    if case["full"]:
        layer += [(h,), (h,), (33,)]           # norms, and a short vector that leaves what follows unaligned
    return layer * case["layers"]


def _prepare_clip(case, seed, g):
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    dtype, out = _DTYPES[case["dtype"]], _DTYPES[case["out"]]
    flat = torch.empty(sum(sizes), device="cuda", dtype=dtype)
    into = torch.empty(sum(sizes), device="cuda", dtype=out)
    std = 1e-3 * case["scale"]
    for at in range(0, flat.numel(), 1 << 26):
        part = flat[at:at + (1 << 26)]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(std))
    grads = [p.view(s) for p, s in zip(flat.split(sizes), shapes)]
    dest = [p.view(s) for p, s in zip(into.split(sizes), shapes)]
    groups = case["slots"] if case["per_slot"] else 1
    if case["per_slot"]:         # the policies' gradients are not of one size
        louder = 0.25 * 16 ** torch.rand(groups, device="cuda", generator=g)
        for grad in grads:
            grad.mul_(louder.to(dtype)[:, None, None])
    state = {"case": case, "grads": grads, "into": into, "out": dest,
             "max_norm": case["bound"] * 1e-3 * math.sqrt(sum(sizes) / groups)}
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_linear(case, seed, g) if case["op"] == "linear" else _prepare_clip(case, seed, g)


# ------------------------------------------------------------------------------------- plain forms
def _plain_linear(state):
    case, scale = state["case"], state["scale"]
    x, w, a, b = (state[i].detach().float() for i in ("x", "weight", "a", "b"))
    dtype = state["x"].dtype
    y = x @ w.t()
    mid = {}
    for s, at in state["rows"].items():
        mid[s] = x[at] @ a[s].t()
        y[at] += scale * (mid[s] @ b[s].t())
    out = {"y": y.to(dtype)}
    if case["train"]:
        dy = state["dy"].float()
        dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
        for s, at in state["rows"].items():
            du = scale * (dy[at] @ b[s])
            dx[at] += du @ a[s]
            da[s] = du.t() @ x[at]
            db[s] = scale * (dy[at].t() @ mid[s])
        out.update(dx=dx.to(dtype), da=da.to(dtype), db=db.to(dtype))
    return out


def _plain_clip(state):
    case = state["case"]
    sums = []
    for grad in state["grads"]:
        rows = grad.view(grad.shape[0] if case["per_slot"] else 1, -1).double()
        sums.append((rows * rows).sum(dim=1))
    norm = torch.sqrt(torch.stack(sums).sum(dim=0)) / case["scale"]
    factor = (torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0) / case["scale"]).float()
    for grad, to in zip(state["grads"], state["out"]):
        rows = grad.view(factor.shape[0], -1)
        to.view(factor.shape[0], -1).copy_(rows.float() * factor[:, None])
    norm = norm.float()
    return {"norm": norm if case["per_slot"] else norm[0], "grads": state["into"]}


# ---------------------------------------------------------------------------------- the two forms
def _own_linear(state):
    from bridge_b200.ops import adapter_linear

    x, a, b = state["x"], state["a"], state["b"]
    y = adapter_linear(x, state["weight"], a, b, state["rows"], state["scale"])
    out = {"y": y.detach()}
    if state["case"]["train"]:
        out["dx"], out["da"], out["db"] = torch.autograd.grad(y, (x, a, b), state["dy"])
    return out


def _own_clip(state):
    from bridge_b200.ops import clip_grad_norm

    case = state["case"]
    norm = clip_grad_norm(state["grads"], state["max_norm"], per_slot=case["per_slot"], grad_scale=case["scale"],
                          out=state["out"])
    return {"norm": norm, "grads": state["into"]}


def run(state):
    if state["case"]["op"] == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    return _own_clip(state) if own else _plain_clip(state)


def work(case):
    if case["op"] == "clip":
        width = {"bf16": 2, "f16": 2, "f32": 4}
        n = sum(math.prod(s) for s in _shapes(case))
        # one square and sum, one product a value
        return {"bytes": n * (width[case["dtype"]] + width[case["out"]]), "flops": 3 * n}
    t, k, n, s, r = (case[i] for i in ("rows", "k", "n", "slots", "rank"))
    shared, low, adapters = 2 * t * k * n, 2 * t * r * (k + n), min(s, case["requests"]) * r * (k + n)
    if case["train"]:
        return {"bytes": 2 * (2 * t * (k + n) + n * k + adapters + s * r * (k + n)), "flops": 2 * shared + 3 * low}
    return {"bytes": 2 * (t * (k + n) + n * k + adapters), "flops": shared + low}


# ----------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in 64 bits: each request through its own merged weight ``W + scale B A``."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        groups = case["slots"] if case["per_slot"] else 1
        total = torch.zeros(groups, dtype=torch.float64, device="cuda")
        for grad in state["grads"]:
            total += torch.linalg.vector_norm(grad.double().reshape(groups, -1), dim=1) ** 2
        norm = total.sqrt() / case["scale"]
        factor = torch.where(norm + 1e-6 > state["max_norm"], state["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
        parts = [(grad.double().reshape(groups, -1) * (factor / case["scale"])[:, None]).reshape(-1)
                 for grad in state["grads"]]
        return {"norm": norm if case["per_slot"] else norm[0], "grads": torch.cat(parts)}
    x, w, a, b = (state[i].detach().double() for i in ("x", "weight", "a", "b"))
    scale, cu, slots = state["scale"], state["cu"], state["slots"]
    y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    if case["train"]:
        dy, dx = state["dy"].double(), torch.empty_like(x)
        da, db = torch.zeros_like(a), torch.zeros_like(b)
    for s in sorted(set(slots)):
        mine = [i for i, t in enumerate(slots) if t == s]
        merged = w if s < 0 else w + scale * (b[s] @ a[s])
        outer = 0.0
        for i in mine:
            at = slice(cu[i], cu[i + 1])
            y[at] = x[at] @ merged.t()
            if case["train"]:
                dx[at] = dy[at] @ merged
                outer = outer + dy[at].t() @ x[at]
        if case["train"] and s >= 0:         # the merged weight's gradient, taken to its two factors
            da[s], db[s] = scale * (b[s].t() @ outer), scale * (outer @ a[s].t())
    return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else {"y": y}
