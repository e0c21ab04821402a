"""Attention over [B, H, T, D] views, forward and recomputing backward.

``out_i = sum_j softmax_j(sm_scale q_i . k_j) v_j`` over the keys that are valid
for row i: ``j <= i`` when causal, and tokens that the [B, T] padding mask
keeps.  A token that the mask removes is neither a query nor a key: its rows of
the output and of every gradient are 0, and what its rows of the inputs hold
(NaN included) reaches no other row.  Key heads are shared by ``Hq / Hkv``
query heads, as in ``attn_kl_align``.

This is the attention that LinearARD's capture hook runs beside recording q, k
and v (``train.py:116-146``).  It reads the views that the attention layer
holds, and lays its output and gradients out as the tensor they belong to
([B, T, H, D] memory for a transposed projection), so that no copy stands
before or after it.  The backward keeps no [T, T] map: it recomputes the
probabilities from q, k and the row log-sum-exp (``lkl_attn_forward`` /
``lkl_attn_backward``).  Results are reproducible bit for bit.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .._marshal import on_device, once_when_recorded, raw_stream, same_as_saved
from ..attention_KL._common import (_DT, _MASK_DT, SUPPORTED_HEAD_DIMS, TC_HEAD_DIMS, check_lse,
                                    prepare_mask, scale_of)

__all__ = ["attn", "attn_forward", "attn_backward", "AttnFn"]

# element strides (b, h, t) of the tensors of a call, in the library's order
_Strides4, _Strides8 = ctypes.c_int64 * 12, ctypes.c_int64 * 24


def _check(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        assert isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor"
        assert t.is_cuda, "q/k/v must be on CUDA"
        assert t.dtype in _DT, f"{name} dtype supports only fp16/bf16"
        assert t.ndim == 4, f"{name} shape must be [B,H,T,D]"
        assert t.stride(-1) == 1, f"{name} last-dim stride must be 1"
    assert q.dtype == k.dtype == v.dtype, "q/k/v dtype must match"
    assert q.device == k.device == v.device, "q/k/v must be on the same device"
    (B, Hq, T, D), (Bk, Hkv, Tk, Dk) = q.shape, k.shape
    assert v.shape == k.shape, "k/v shape must match"
    assert (B, T, D) == (Bk, Tk, Dk), "q/k B/T/D must match"
    assert Hkv > 0 and Hq > 0, "there must be a head"
    assert Hq % Hkv == 0, "Hq must be divisible by Hkv"
    assert D in SUPPORTED_HEAD_DIMS, "head_dim is not in the supported set"


def _problem(q, k, causal, mask_dtype, sm_scale):
    B, Hq, T, D = q.shape
    sc = scale_of(sm_scale, D, "sm_scale")
    # normal numbers of single precision, also when multiplied by log2(e)
    assert 2.0 ** -126 <= sc < 2.0 ** 127, "sm_scale must be positive"
    return _lib.LKLAttnProblem(B, Hq, k.shape[1], T, D, _DT[q.dtype], 1 if causal else 0,
                               mask_dtype, sc)


def _strides(t):
    """Element strides (b, h, t); a dim of size 1 gets one that any path can read."""
    (b, h, n, _), (B, H, T, D) = t.stride(), t.shape
    return (b if B != 1 else D, h if H != 1 else D, n if T != 1 else D)


def _readable(t):
    """(tensor, strides): t itself, or a contiguous copy where the tensor-core
    kernels cannot read it in place (the CUDA-core ones could, many times slower)."""
    b, h, n, unit = t.stride()
    B, H, T, D = t.shape
    b, h, n = b if B != 1 else D, h if H != 1 else D, n if T != 1 else D    # as in _strides
    if unit == 1 and (D not in TC_HEAD_DIMS or (b > 0 and h > 0 and n > 0 and not (b | h | n) % 8
                                                and not t.data_ptr() % 16)):
        return t, (b, h, n)
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _strides(t)


def _like(t):
    """(tensor, strides): uninitialised, of t's shape and type, in its order of heads
    and tokens."""
    B, H, T, D = t.shape
    s = t.stride()
    n = H * T * D
    if s == (n, T * D, D, 1) or s == (n, D, H * D, 1):
        return torch.empty_like(t), s[:3]      # dense: keeps the strides
    if s[1] < s[2]:
        return (torch.empty((B, T, H, D), device=t.device, dtype=t.dtype).transpose(1, 2),
                (n, D, H * D))
    return torch.empty((B, H, T, D), device=t.device, dtype=t.dtype), (n, T * D, D)


def _workspace(n, device):
    """(tensor to hold, its address)"""
    if not n:
        return None, None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def _forward(q, k, v, mask, prob):
    """(out, lse) of checked arguments; mask on the device or None."""
    L, dev = _lib.lib(), q.device
    with on_device(dev):
        (rq, sq), (rk, sk), (rv, sv) = _readable(q), _readable(k), _readable(v)
        out, so = _like(rq)
        lse = torch.empty((prob.B, prob.Hq, prob.T), device=dev, dtype=torch.float32)
        ref = ctypes.byref(prob)
        n, ws, at, m = 0, None, None, None
        if mask is not None:
            n, m = L.lkl_attn_forward_workspace_size(ref, 1), mask.data_ptr()
            ws, at = _workspace(n, dev)
        st = L.lkl_attn_forward(rq.data_ptr(), rk.data_ptr(), rv.data_ptr(),
                                _Strides4(*sq, *sk, *sv, *so), m, ref,
                                out.data_ptr(), lse.data_ptr(), at, n, raw_stream(dev))
    _lib.check(st, "lkl_attn_forward")
    return out, lse


def _backward(dout, q, k, v, out, lse, mask, prob):
    L, dev = _lib.lib(), q.device
    with on_device(dev):
        (dq, sdq), (dk, sdk), (dv, sdv) = _like(q), _like(k), _like(v)
        (q, sq), (k, sk), (v, sv), (out, so) = (_readable(t) for t in (q, k, v, out))
        dout, sd = _readable(dout)
        ref = ctypes.byref(prob)
        n = L.lkl_attn_backward_workspace_size(ref, 0 if mask is None else 1)
        ws, at = _workspace(n, dev)
        st = L.lkl_attn_backward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            dout.data_ptr(), _Strides8(*sq, *sk, *sv, *so, *sd, *sdq, *sdk, *sdv),
            None if mask is None else mask.data_ptr(), ref, dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), at, n, raw_stream(dev))
    _lib.check(st, "lkl_attn_backward")
    return dq, dk, dv


def attn_forward(q, k, v, attn_mask=None, causal=True, sm_scale=None):
    """q [B,Hq,T,D], k and v [B,Hkv,T,D] -> (out [B,Hq,T,D], lse [B,Hq,T] fp32).
    Rows that the mask removes have out 0 and lse 0."""
    _check(q, k, v)
    mask, mdt = prepare_mask(attn_mask, q.shape[0], q.shape[2], q.device)
    return _forward(q, k, v, mask, _problem(q, k, causal, mdt, sm_scale))


def attn_backward(dout, q, k, v, out, lse, attn_mask=None, causal=True, sm_scale=None):
    """Gradients (dq, dk, dv) of q, k and v, of their types and in their order
    of heads and tokens; out and lse are attn_forward's."""
    _check(q, k, v)
    for name, t in (("dout", dout), ("out", out)):
        assert isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor"
        assert t.shape == q.shape and t.dtype == q.dtype and t.device == q.device, \
            f"{name} must have the shape, dtype and device of q"
    check_lse(lse, q.shape[:3])
    assert lse.device == q.device, "lse must be on the device of q"
    mask, mdt = prepare_mask(attn_mask, q.shape[0], q.shape[2], q.device)
    return _backward(dout, q, k, v, out, lse, mask, _problem(q, k, causal, mdt, sm_scale))


class AttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, prob):
        out, lse = _forward(q, k, v, mask, prob)
        ctx.save_for_backward(q, k, v, out, lse, mask)
        ctx.prob, ctx.kv_shape = prob, k.shape
        return out

    @once_when_recorded
    def backward(ctx, dout):
        q, k, v, out, lse, mask = ctx.saved_tensors
        # strides are read from what came back: a hook may have changed them
        p, dt, dev, shape, kv = ctx.prob, dout.dtype, dout.device, dout.shape, ctx.kv_shape
        same_as_saved(q, shape, dt, dev)
        same_as_saved(k, kv, dt, dev)
        same_as_saved(v, kv, dt, dev)
        same_as_saved(out, shape, dt, dev)
        lse = same_as_saved(lse, shape[:3], torch.float32, dev).contiguous()
        if mask is not None:
            assert _MASK_DT.get(mask.dtype) == p.mask_dtype, "a saved mask came back as another type"
            mask = same_as_saved(mask, (p.B, p.T), mask.dtype, dev).contiguous()
        dq, dk, dv = _backward(dout, q, k, v, out, lse, mask, p)
        return dq, dk, dv, None, None


def attn(q, k, v, attn_mask=None, causal=True, sm_scale=None):
    """Attention with gradients for q, k and v.  q: [B,Hq,T,D], k and v:
    [B,Hkv,T,D], fp16 or bf16 on CUDA, any strides with a last one of 1 (copied
    where they are not multiples of 8 elements); attn_mask: [B,T], nonzero =
    token, or None; sm_scale: default 1/sqrt(D).  Returns [B,Hq,T,D] in the
    memory order of q."""
    _check(q, k, v)
    mask, mdt = prepare_mask(attn_mask, q.shape[0], q.shape[2], q.device)
    return AttnFn.apply(q, k, v, mask, _problem(q, k, causal, mdt, sm_scale))
