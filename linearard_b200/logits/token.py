"""Log probabilities of given tokens, with entropy and top alternatives.

``token_logprobs(logits, targets, top_k=0, ignore_index=-100)`` reads the
logits once and never writes a [.., V] tensor of probabilities.  It takes views
such as ``logits[:, :-1]`` as they are.  ``-logprob.sum()`` is the next-token
loss; the gradients of logprob and entropy flow to the logits
(``lkl_token_logprobs`` / ``lkl_token_logprobs_backward``).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._marshal import on_device, once_when_recorded, raw_stream, same_as_saved
from ._common import check_logits, rows_of, saved_rows

__all__ = ["token_logprobs", "TokenLogprobs", "TokenLogprobsFn", "MAX_TOP_K"]

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    """fp32 [B, T] each; the alternatives [B, T, top_k] (None without them)."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def _forward(logits, rows, targets, top_k, ignore_index, keep=False):
    """(logprob, entropy, lse, top_logprobs, top_indices) of checked arguments.
    keep: lse for the backward, [2, ...]: its fp32 value and what that lacks."""
    dev, shape = logits.device, targets.shape
    with on_device(dev):
        # tensors of their own: views of one could not be changed in place
        logprob = torch.empty(shape, device=dev, dtype=torch.float32)
        entropy = torch.empty_like(logprob)
        if keep:
            lse = torch.empty((2, *shape), device=dev, dtype=torch.float32)
            rows.lse_low = lse.data_ptr() + 4 * logprob.numel()
        else:
            lse = torch.empty_like(logprob)
        top_v = top_i = None
        if top_k:
            top_v = torch.empty((*shape, top_k), device=dev, dtype=torch.float32)
            top_i = torch.empty((*shape, top_k), device=dev, dtype=torch.int64)
        st = _lib.lib().lkl_token_logprobs(
            logits.data_ptr(), ctypes.byref(rows), targets.data_ptr(), ignore_index, top_k,
            logprob.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
            top_v.data_ptr() if top_k else None, top_i.data_ptr() if top_k else None,
            raw_stream(dev))
    _lib.check(st, "lkl_token_logprobs")
    return logprob, entropy, lse, top_v, top_i


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, targets, top_k: int, ignore_index: int):
        logprob, entropy, lse, top_v, top_i = _forward(logits, rows, targets, top_k, ignore_index,
                                                       keep=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, lse, entropy)
        ctx.shape, ctx.dtype, ctx.device = logits.shape, logits.dtype, logits.device
        ctx.seen, ctx.ignore_index = (rows, logits.stride()), ignore_index
        if top_k:
            ctx.mark_non_differentiable(top_v, top_i)
        return logprob, entropy, top_v, top_i

    @once_when_recorded
    def backward(ctx, d_logprob, d_entropy, _top_v, _top_i):
        if d_logprob is None and d_entropy is None:
            return None, None, None, None, None
        logits, targets, lse, entropy = ctx.saved_tensors
        dev, shape = ctx.device, ctx.shape[:-1]
        with on_device(dev):
            logits, rows = saved_rows(logits, ctx.shape, ctx.dtype, dev, ctx.seen)
            targets = same_as_saved(targets, shape, torch.int64, dev).contiguous()
            lse = same_as_saved(lse, (2, *shape), torch.float32, dev).contiguous()
            rows.lse_low = lse.data_ptr() + 4 * entropy.numel()
            entropy = same_as_saved(entropy, shape, torch.float32, dev).contiguous()
            g, h = (None if d is None else d.to(torch.float32).contiguous()
                    for d in (d_logprob, d_entropy))
            dx = torch.empty(ctx.shape, device=dev, dtype=ctx.dtype)
            st = _lib.lib().lkl_token_logprobs_backward(
                logits.data_ptr(), ctypes.byref(rows), targets.data_ptr(), ctx.ignore_index,
                lse.data_ptr(), entropy.data_ptr(), None if g is None else g.data_ptr(),
                None if h is None else h.data_ptr(), dx.data_ptr(), raw_stream(dev))
        _lib.check(st, "lkl_token_logprobs_backward")
        return dx, None, None, None, None


def token_logprobs(logits, targets, top_k=0, ignore_index=-100) -> TokenLogprobs:
    """logits: [B,T,V] (or [N,V]) fp16, bf16 or fp32 on CUDA, last stride 1;
    targets: int64 [B,T] (or [N]).  logprob is 0 where the target is
    ignore_index and NaN where it is any other number outside [0, V).
    top_k: up to 32 alternatives, largest first, equal logits by the lowest
    index.  logprob and entropy carry gradients to the logits; the
    alternatives carry none.  logprob may be changed in place; the backward needs
    entropy as it is (autograd raises where it was changed)."""
    check_logits(logits)
    assert isinstance(targets, torch.Tensor), "targets must be a torch.Tensor"
    assert targets.device == logits.device, "targets must be on the device of the logits"
    assert targets.dtype == torch.int64, "targets must be int64"
    assert targets.shape == logits.shape[:-1], "targets shape must be that of the logits' rows"
    assert isinstance(top_k, int) and 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]), \
        "top_k must be from 0 to min(V, 32)"
    assert isinstance(ignore_index, int) and -2 ** 63 <= ignore_index < 2 ** 63, \
        "ignore_index must be an integer of 64 bits"
    rows, targets = rows_of(logits), targets.contiguous()
    # a dual tensor does not require grad: the function refuses it, its tangent is not lost
    if (logits.requires_grad and torch.is_grad_enabled()
            or forward_ad.unpack_dual(logits).tangent is not None):
        return TokenLogprobs(*TokenLogprobsFn.apply(logits, rows, targets, top_k, ignore_index))
    logprob, entropy, _, top_v, top_i = _forward(logits, rows, targets, top_k, ignore_index)
    return TokenLogprobs(logprob, entropy, top_v, top_i)
