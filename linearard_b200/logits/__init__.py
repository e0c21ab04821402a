"""Operators over rows of logits: the KL between the two models' distributions
and the log probabilities of given tokens."""
from .kl import LogitsKLAlignFn, logits_kl_align, logits_kl_backward, logits_kl_forward
from .token import MAX_TOP_K, TokenLogprobs, TokenLogprobsFn, token_logprobs

__all__ = ["logits_kl_align", "logits_kl_forward", "logits_kl_backward", "LogitsKLAlignFn",
           "token_logprobs", "TokenLogprobs", "TokenLogprobsFn", "MAX_TOP_K"]
