"""Hot ops: sm_100a CUDA kernels on CUDA tensors, PyTorch formulations on CPU."""

from .activation import swiglu
from .adapter import AdapterRows, adapter_linear, adapter_rows
from .attention import rectangular_causal_attention, tree_attention
from .distill import fused_lm_head_topk_distill, topk_distill_loss
from .gdn import causal_conv1d, chunk_gated_delta_rule
from .grad_norm import clip_grad_norm, global_grad_norm
from .logprob import fused_lm_head_logprob
from .norm import qk_norm_rope, rmsnorm
from .ppo import PPOLossConfig, ppo_loss
from .token_logprob import TokenLogprobs, fused_lm_head_token_logprobs, token_logprobs
