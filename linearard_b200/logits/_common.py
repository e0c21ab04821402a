"""Argument checks and C-ABI marshalling of the logits operators."""
from __future__ import annotations

import torch

from .. import _lib
from .._marshal import same_as_saved

_DT = {torch.float16: _lib.LKL_F16, torch.bfloat16: _lib.LKL_BF16, torch.float32: _lib.LKL_F32}


def check_logits(x, name="logits"):
    assert isinstance(x, torch.Tensor), f"{name} must be a torch.Tensor"
    assert x.is_cuda, f"{name} must be on CUDA"
    assert x.dtype in _DT, f"{name} dtype supports only fp16/bf16/fp32"
    assert x.ndim in (2, 3), f"{name} shape must be [B,T,V] or [N,V]"
    assert x.shape[-1] > 0, f"{name} must have a vocabulary"
    assert x.stride(-1) == 1 or x.shape[-1] == 1, f"{name} last-dim stride must be 1"


def rows_of(x) -> _lib.LKLLogits:
    """The rows of [B, T, V] or [N, V] logits, read in place."""
    if x.ndim == 2:
        return _lib.LKLLogits(1, x.shape[0], x.shape[1], 0, x.stride(0), _DT[x.dtype])
    return _lib.LKLLogits(*x.shape, *x.stride()[:2], _DT[x.dtype])


def saved_rows(x, shape, dtype, device, seen):
    """(tensor, its rows) of logits that autograd kept for a backward: the strides are
    those that it came back with.  seen: the forward's (rows, strides)."""
    same_as_saved(x, shape, dtype, device)
    strides = x.stride()
    if strides == seen[1]:
        return x, seen[0]
    if strides[-1] != 1 and shape[-1] != 1:
        x = x.contiguous()
    return x, rows_of(x)
