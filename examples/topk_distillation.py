"""Distil a teacher policy into a student from the teacher's top log-probs.

Every step runs the teacher over a batch of sequences, keeps its ``--top-k`` likeliest next tokens per
position, trains the student on the divergence from them, and scores the student's log-probs of the
teacher's first choices::

    python examples/topk_distillation.py                       # tiny models, on the GPU if there is one
    python examples/topk_distillation.py --model qwen3_4b --layers 4 --rows 2048 --top-k 64
"""

from __future__ import annotations

import argparse
import os
import sys
from dataclasses import replace

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from bridge_b200.engine.optim import AdamWConfig, MixedPrecisionAdamW  # noqa: E402
from bridge_b200.models import build_model, get_config  # noqa: E402
from bridge_b200.ops import fused_lm_head_token_logprobs  # noqa: E402
from bridge_b200.rl import distill_loss, teacher_alternatives  # noqa: E402


def run(model: str = "tiny", layers: int | None = None, rows: int = 128, top_k: int = 16, steps: int = 8,
        lr: float = 2e-3, tail: bool = True, temperature: float = 1.0, device: str | None = None,
        seed: int = 0) -> list[dict]:
    """Returns one record per step: the loss, the student's entropy and its mean log-prob of the teacher's first
    choice."""
    device = device or ("cuda" if torch.cuda.is_available() else "cpu")
    cfg = get_config(model, **({"num_layers": layers} if layers else {}))
    # random weights, drawn wider for the teacher: its next-token distributions are far from flat
    teacher = build_model(replace(cfg, init_std=4 * cfg.init_std), device=device, seed=seed + 1)
    student = build_model(cfg, device=device, seed=seed + 2)
    optimizer = MixedPrecisionAdamW(student, AdamWConfig(lr=lr))
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, cfg.vocab_size, (rows,), generator=g).to(device)
    positions = torch.arange(rows, device=device)
    history = []
    for _ in range(steps):
        with torch.no_grad():
            top_ids, top_logp = teacher_alternatives(teacher, teacher(ids, positions, rows), top_k=top_k,
                                                     temperature=temperature)
        hidden = student(ids, positions, rows)
        loss, _ = distill_loss(student, hidden, top_ids, top_logp, denom=float(rows), temperature=temperature,
                               tail=tail)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad()
        scores = fused_lm_head_token_logprobs(hidden.detach(), student.head_weight, top_ids[:, 0], temperature)
        history.append({"loss": float(loss.detach()), "entropy": float(scores.entropy.mean()),
                        "first_choice_logp": float(scores.logp.mean())})
    return history


def main(argv=None) -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--model", default="tiny")
    p.add_argument("--layers", type=int, default=None, help="cut the preset to this many layers")
    p.add_argument("--rows", type=int, default=128, help="tokens per step")
    p.add_argument("--top-k", type=int, default=16)
    p.add_argument("--steps", type=int, default=8)
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--no-tail", action="store_true", help="renormalise the teacher's entries instead of a tail class")
    a = p.parse_args(argv)
    for i, r in enumerate(run(a.model, a.layers, a.rows, a.top_k, a.steps, a.lr, not a.no_tail, a.temperature)):
        print(f"step {i}: loss {r['loss']:.4f}  entropy {r['entropy']:.3f}  "
              f"first choice log-prob {r['first_choice_logp']:.3f}", flush=True)


if __name__ == "__main__":
    main()
