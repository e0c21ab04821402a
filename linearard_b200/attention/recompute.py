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
from ..attention_KL._common import (_DT, SUPPORTED_HEAD_DIMS, TC_HEAD_DIMS, check_lse,
                                    prepare_mask, ptr, scale_of, stream_of)

__all__ = ["attn", "attn_forward", "attn_backward", "AttnFn"]


def _check(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        assert isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor"
        assert t.is_cuda, "q/k/v must be on CUDA"
        assert t.dtype in (torch.float16, torch.bfloat16), f"{name} dtype supports only fp16/bf16"
        assert t.ndim == 4, f"{name} shape must be [B,H,T,D]"
        assert t.stride(-1) == 1, f"{name} last-dim stride must be 1"
    assert q.dtype == k.dtype == v.dtype, "q/k/v dtype must match"
    assert q.device == k.device == v.device, "q/k/v must be on the same device"
    assert k.shape == v.shape, "k/v shape must match"
    assert (k.shape[0], k.shape[2], k.shape[3]) == (q.shape[0], q.shape[2], q.shape[3]), \
        "q/k B/T/D must match"
    assert k.shape[1] > 0 and q.shape[1] > 0, "there must be a head"
    assert q.shape[1] % k.shape[1] == 0, "Hq must be divisible by Hkv"
    assert q.shape[3] in SUPPORTED_HEAD_DIMS, "head_dim is not in the supported set"


def _scale(sm_scale, D):
    sc = scale_of(sm_scale, D, "sm_scale")
    assert 0.0 < sc < float("inf"), "sm_scale must be positive"
    return sc


def _problem(q, k, causal, mask_dtype, sm_scale):
    B, Hq, T, D = q.shape
    return _lib.LKLAttnProblem(B=B, Hq=Hq, Hkv=k.shape[1], T=T, D=D, dtype=_DT[q.dtype],
                               causal=1 if causal else 0, mask_dtype=mask_dtype,
                               sm_scale=_scale(sm_scale, D))


def _stride(t):
    """Element strides (b, h, t); a dim of size 1 gets one that any path can read."""
    b, h, n = (t.stride(i) if t.shape[i] != 1 else t.shape[3] for i in range(3))
    return _lib.LKLStrides(b=b, h=h, t=n)


def _readable(t):
    """`t`, or a contiguous copy where the tensor-core kernels cannot read it in
    place (their CUDA-core counterparts could, many times slower)."""
    if t.shape[3] in TC_HEAD_DIMS:
        s = _stride(t)
        if (t.data_ptr() % 16 or t.stride(3) != 1
                or any(x <= 0 or x % 8 for x in (s.b, s.h, s.t))):
            return t.clone(memory_format=torch.contiguous_format)
    return t if t.stride(3) == 1 else t.contiguous()


def _like(t):
    """An uninitialised tensor of t's shape and type, in its order of heads and tokens."""
    B, H, T, D = t.shape
    if t.stride(1) < t.stride(2):
        return torch.empty((B, T, H, D), device=t.device, dtype=t.dtype).transpose(1, 2)
    return torch.empty((B, H, T, D), device=t.device, dtype=t.dtype)


def _strides(*tensors):
    return (_lib.LKLStrides * len(tensors))(*[_stride(t) for t in tensors])


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def attn_forward(q, k, v, attn_mask=None, causal=True, sm_scale=None):
    """q [B,Hq,T,D], k and v [B,Hkv,T,D] -> (out [B,Hq,T,D], lse [B,Hq,T] fp32).
    Rows that the mask removes have out 0 and lse 0."""
    _check(q, k, v)
    B, Hq, T, _ = q.shape
    mask, mdt = prepare_mask(attn_mask, B, T, q.device)
    prob = _problem(q, k, causal, mdt, sm_scale)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        q, k, v = _readable(q), _readable(k), _readable(v)
        out = _like(q)
        lse = torch.empty((B, Hq, T), device=q.device, dtype=torch.float32)
        n = int(L.lkl_attn_forward_workspace_size(ctypes.byref(prob), 1 if mask is not None else 0))
        ws = _workspace(n, q.device)
        st = L.lkl_attn_forward(ptr(q), ptr(k), ptr(v), _strides(q, k, v, out), ptr(mask),
                                ctypes.byref(prob), ptr(out), ptr(lse), ptr(ws), n,
                                stream_of(q.device))
    _lib.check(st, "lkl_attn_forward")
    return out, lse


def attn_backward(dout, q, k, v, out, lse, attn_mask=None, causal=True, sm_scale=None):
    """Gradients (dq, dk, dv) of q, k and v, of their types and in their order
    of heads and tokens; out and lse are attn_forward's."""
    _check(q, k, v)
    for name, t in (("dout", dout), ("out", out)):
        assert isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor"
        assert t.shape == q.shape and t.dtype == q.dtype and t.device == q.device, \
            f"{name} must have the shape, dtype and device of q"
    B, Hq, T, _ = q.shape
    check_lse(lse, (B, Hq, T))
    assert lse.device == q.device, "lse must be on the device of q"
    mask, mdt = prepare_mask(attn_mask, B, T, q.device)
    prob = _problem(q, k, causal, mdt, sm_scale)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        dq, dk, dv = _like(q), _like(k), _like(v)
        q, k, v, out, dout = (_readable(t) for t in (q, k, v, out, dout))
        n = int(L.lkl_attn_backward_workspace_size(ctypes.byref(prob),
                                                   1 if mask is not None else 0))
        ws = _workspace(n, q.device)
        st = L.lkl_attn_backward(ptr(q), ptr(k), ptr(v), ptr(out), ptr(lse), ptr(dout),
                                 _strides(q, k, v, out, dout, dq, dk, dv), ptr(mask),
                                 ctypes.byref(prob), ptr(dq), ptr(dk), ptr(dv), ptr(ws), n,
                                 stream_of(q.device))
    _lib.check(st, "lkl_attn_backward")
    return dq, dk, dv


class AttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, attn_mask, causal: bool, sm_scale):
        _check(q, k, v)
        mask, _ = prepare_mask(attn_mask, q.shape[0], q.shape[2], q.device)
        out, lse = attn_forward(q, k, v, mask, causal, sm_scale)
        ctx.save_for_backward(q, k, v, out, lse, mask)
        ctx.causal, ctx.sm_scale = causal, sm_scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, mask = ctx.saved_tensors
        dq, dk, dv = attn_backward(dout, q, k, v, out, lse, mask, ctx.causal, ctx.sm_scale)
        return dq, dk, dv, None, None, None


def attn(q, k, v, attn_mask=None, causal=True, sm_scale=None):
    """Attention with gradients for q, k and v.  q: [B,Hq,T,D], k and v:
    [B,Hkv,T,D], fp16 or bf16 on CUDA, any strides with a last one of 1 (copied
    where they are not multiples of 8 elements); attn_mask: [B,T], nonzero =
    token, or None; sm_scale: default 1/sqrt(D).  Returns [B,Hq,T,D] in the
    memory order of q."""
    return AttnFn.apply(q, k, v, attn_mask, causal, sm_scale)
