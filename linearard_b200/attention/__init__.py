"""The attention of the distillation step, with a backward pass that recomputes
the probabilities: ``attn(q, k, v, attn_mask=None, causal=True, sm_scale=None)``.
"""
from .recompute import AttnFn, attn, attn_backward, attn_forward

__all__ = ["attn", "attn_forward", "attn_backward", "AttnFn"]
