"""KL between the teacher's and the student's logits.

``logits_kl_align(s_logits, t_logits, attn_mask=None, temperature=1.0)`` returns
the 0-d fp32 **sum** over the rows that the mask keeps of
``KL(softmax(t / temperature) || softmax(s / temperature))``; the caller
divides, as with ``attn_kl_align``.  This is the ``lam_l`` term of the training
loop (``train.py:413-423``) without its [B, T, V] tensors of log probabilities:
the forward reads both logits once, the backward once more
(``lkl_logits_kl_forward`` / ``lkl_logits_kl_backward``).
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .._marshal import on_device, once_when_recorded, raw_stream, same_as_saved
from ..attention_KL._common import _MASK_DT, prepare_mask
from ._common import check_logits, rows_of, saved_rows

__all__ = ["logits_kl_align", "logits_kl_forward", "logits_kl_backward", "LogitsKLAlignFn"]


def _check(s, t, temperature):
    check_logits(s, "s_logits")
    check_logits(t, "t_logits")
    assert s.shape == t.shape, "student/teacher logits shape must match"
    assert s.dtype == t.dtype, "student/teacher logits dtype must match"
    assert s.device == t.device, "student/teacher must be on the same device"
    assert isinstance(temperature, (float, int)), "temperature must be a scalar"
    # single precision has to hold the temperature and what it divides by
    assert 1e-30 < temperature < 1e30, "temperature must be positive"


def _mask(attn_mask, s):
    if attn_mask is None:
        return prepare_mask(None, 0, 0, s.device)
    assert isinstance(attn_mask, torch.Tensor), "attn_mask must be a torch.Tensor"
    assert attn_mask.shape == s.shape[:-1], "attn_mask shape must be that of the logits' rows"
    mask = attn_mask.contiguous()
    mask = mask[None] if s.ndim == 2 else mask
    return prepare_mask(mask, mask.shape[0], mask.shape[1], s.device)


def _forward(s, t, mask, mdt, temperature, rows, keep=False):
    """(loss, lse_s, lse_t).  keep: for the backward, one tensor [4, ...] in lse_s: the
    student's log-sum-exp, what its fp32 value lacks, and the teacher's two."""
    dev, shape = s.device, s.shape[:-1]
    L = _lib.lib()
    with on_device(dev):
        if keep:
            lse_s, lse_t = torch.empty((4, *shape), device=dev, dtype=torch.float32), None
            at_s, at_t = _kept(lse_s, rows)
        else:
            lse_s = torch.empty(shape, device=dev, dtype=torch.float32)
            lse_t = torch.empty_like(lse_s)
            at_s, at_t = lse_s.data_ptr(), lse_t.data_ptr()
        loss = torch.empty((), device=dev, dtype=torch.float32)
        rs, rt = ctypes.byref(rows[0]), ctypes.byref(rows[1])
        n = L.lkl_logits_kl_workspace_size(rs)
        ws = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)
        st = L.lkl_logits_kl_forward(s.data_ptr(), rs, t.data_ptr(), rt,
                                     None if mask is None else mask.data_ptr(), mdt, temperature,
                                     at_s, at_t, loss.data_ptr(), ws.data_ptr(), n,
                                     raw_stream(dev))
    _lib.check(st, "lkl_logits_kl_forward")
    return loss, lse_s, lse_t


def _kept(lse, rows):
    """Addresses of the two log-sum-exps in a [4, ...] tensor; the rows learn those of
    what their fp32 values lack."""
    at, n = lse.data_ptr(), lse.numel()     # a quarter of n elements of 4 bytes each
    rows[0].lse_low, rows[1].lse_low = at + n, at + 3 * n
    return at, at + 2 * n


def _backward(s, t, at_s, at_t, mask, mdt, temperature, rows, dloss):
    """at_s, at_t: addresses of the log-sum-exps."""
    dev = s.device
    with on_device(dev):
        ds = torch.empty(s.shape, device=dev, dtype=s.dtype)
        st = _lib.lib().lkl_logits_kl_backward(
            s.data_ptr(), ctypes.byref(rows[0]), t.data_ptr(), ctypes.byref(rows[1]),
            None if mask is None else mask.data_ptr(), mdt, temperature, at_s, at_t,
            None if dloss is None else dloss.data_ptr(), ds.data_ptr(), raw_stream(dev))
    _lib.check(st, "lkl_logits_kl_backward")
    return ds


def logits_kl_forward(s_logits, t_logits, attn_mask=None, temperature=1.0):
    """(loss 0-d fp32, lse_s, lse_t fp32 of the rows' shape: the log-sum-exp of
    logits / temperature, 0 where the mask removes the row)."""
    _check(s_logits, t_logits, temperature)
    mask, mdt = _mask(attn_mask, s_logits)
    return _forward(s_logits, t_logits, mask, mdt, float(temperature),
                    (rows_of(s_logits), rows_of(t_logits)))


def logits_kl_backward(s_logits, t_logits, lse_s, lse_t, attn_mask=None, temperature=1.0,
                       dloss=None):
    """Gradient of the student's logits, contiguous, of their type.  dloss: a
    device fp32 scalar, default 1."""
    _check(s_logits, t_logits, temperature)
    dev, shape = s_logits.device, tuple(s_logits.shape[:-1])
    for z in (lse_s, lse_t):
        assert isinstance(z, torch.Tensor) and tuple(z.shape) == shape, \
            "lse shape must be that of the logits' rows"
        assert z.dtype == torch.float32 and z.is_contiguous() and z.device == dev, \
            "lse must be contiguous float32 on the device of the logits"
    if dloss is not None:
        assert isinstance(dloss, torch.Tensor) and dloss.numel() == 1 and dloss.device == dev \
            and dloss.dtype == torch.float32, "dloss must be a float32 scalar on the device"
    mask, mdt = _mask(attn_mask, s_logits)
    return _backward(s_logits, t_logits, lse_s.data_ptr(), lse_t.data_ptr(), mask, mdt,
                     float(temperature), (rows_of(s_logits), rows_of(t_logits)), dloss)


class LogitsKLAlignFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s_logits, t_logits, mask, mdt, temperature, rows):
        loss, lse, _ = _forward(s_logits, t_logits, mask, mdt, temperature, rows, keep=True)
        ctx.save_for_backward(s_logits, t_logits, lse, mask)
        ctx.mdt, ctx.temperature = mdt, temperature
        ctx.seen = (rows[0], s_logits.stride()), (rows[1], t_logits.stride())
        ctx.shape, ctx.dtype, ctx.device = s_logits.shape, s_logits.dtype, s_logits.device
        return loss

    @once_when_recorded
    def backward(ctx, dloss):
        s_logits, t_logits, lse, mask = ctx.saved_tensors
        shape, dt, dev = ctx.shape, ctx.dtype, ctx.device
        lse = same_as_saved(lse, (4, *shape[:-1]), torch.float32, dev).contiguous()
        if mask is not None:
            assert _MASK_DT.get(mask.dtype) == ctx.mdt, "a saved mask came back as another type"
            rows = shape[:-1] if len(shape) == 3 else (1, shape[0])
            mask = same_as_saved(mask, rows, mask.dtype, dev).contiguous()
        s_logits, s_rows = saved_rows(s_logits, shape, dt, dev, ctx.seen[0])
        t_logits, t_rows = saved_rows(t_logits, shape, dt, dev, ctx.seen[1])
        rows = (s_rows, t_rows)
        ds = _backward(s_logits, t_logits, *_kept(lse, rows), mask, ctx.mdt, ctx.temperature,
                       rows, dloss.to(torch.float32))
        return ds, None, None, None, None, None      # the teacher gets no gradient


def logits_kl_align(s_logits, t_logits, attn_mask=None, temperature=1.0):
    """s_logits, t_logits: [B,T,V] (or [N,V]), fp16, bf16 or fp32 of one type, last
    stride 1, read in place; attn_mask: [B,T] (or [N]), nonzero = kept, or None.
    Gradients flow to the student's logits only."""
    _check(s_logits, t_logits, temperature)
    mask, mdt = _mask(attn_mask, s_logits)
    return LogitsKLAlignFn.apply(s_logits, t_logits, mask, mdt, float(temperature),
                                 (rows_of(s_logits), rows_of(t_logits)))
