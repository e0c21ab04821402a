"""B200 (sm_100a) attention-relation KL loss of LinearARD, with the attention and
the logits operators of its distillation step.

The compute lives in ``liblinearard_b200.so`` (C ABI, ``include/linearard_b200.h``);
this package is the PyTorch-facing mirror of LinearARD's ``kernels/attention_KL``.
"""
from .attention_KL import (AttnKLAlignFn, attn_kl_align, attn_kl_forward, kl_backward,
                           kl_forward, lse_stats)
from .attention import AttnFn, attn, attn_backward, attn_forward
from .logits import (logits_kl_align, logits_kl_backward, logits_kl_forward, token_logprobs)

__all__ = ["AttnKLAlignFn", "attn_kl_align", "attn_kl_forward", "lse_stats", "kl_forward",
           "kl_backward", "attn", "attn_forward", "attn_backward", "AttnFn", "logits_kl_align",
           "logits_kl_forward", "logits_kl_backward", "token_logprobs"]
__version__ = "0.1.0"
