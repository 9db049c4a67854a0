"""Distilling a teacher policy into a student through the teacher's likeliest tokens.

The teacher is run once per batch and kept as ``top_k`` token ids with log-probs per supervised row
(:func:`teacher_alternatives`, no gradient); the student's loss on the same rows is the divergence from
them (:func:`distill_loss`).  Both go through the model's LM head a chunk of rows at a time, under tensor
parallelism too, so no ``[rows, vocab]`` tensor outlives a call.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ..ops.distill import fused_lm_head_topk_distill
from ..ops.token_logprob import fused_lm_head_token_logprobs


@torch.no_grad()
def teacher_alternatives(model, hidden_rows: Tensor, *, top_k: int, temperature: Tensor | float = 1.0,
                         chunk_rows: int = 4096) -> tuple[Tensor, Tensor]:
    """``(ids [U, top_k], log-probs)`` of the teacher's likeliest next tokens at ``hidden_rows [U, H]``."""
    r = fused_lm_head_token_logprobs(hidden_rows, model.head_weight, None, temperature, top_k=top_k,
                                     with_entropy=False, vocab_start=model.vocab_start, tp_group=model.tp_group,
                                     chunk_rows=chunk_rows)
    return r.top_ids, r.top_logp


def distill_loss(model, hidden_rows: Tensor, teacher_ids: Tensor, teacher_logp: Tensor, *, denom: float,
                 weights: Tensor | None = None, temperature: Tensor | float = 1.0, tail: bool = True,
                 grad_scale: float = 1.0, chunk_rows: int = 4096) -> tuple[Tensor, Tensor]:
    """``(sum_u w_u KL_u / denom, KL [U])`` of the student at ``hidden_rows``; any factor on the loss is
    right; one that ``grad_scale`` announces saves a rounding of the gradients."""
    return fused_lm_head_topk_distill(model.head_input(hidden_rows), model.head_weight, teacher_ids, teacher_logp,
                                      denom=denom, weights=weights, temperature=temperature, tail=tail,
                                      grad_scale=grad_scale, vocab_start=model.vocab_start, tp_group=model.tp_group,
                                      chunk_rows=chunk_rows)
