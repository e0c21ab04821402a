"""Attention and logits operators without a GPU: refusals before any device
work, from Python and through the C ABI, and the scratch sizes."""
import ctypes

import pytest
import torch

from linearard_b200 import _lib
from linearard_b200.attention import attn, attn_forward
from linearard_b200.logits import logits_kl_align, token_logprobs

FAKE, FAKE2, FAKE3, FAKE4 = (ctypes.c_void_p(0x10000 * i) for i in (1, 2, 3, 4))


def prob(**kw):
    d = dict(B=2, Hq=4, Hkv=2, T=300, D=128, dtype=1, causal=1, mask_dtype=3, sm_scale=0.0)
    d.update(kw)
    return _lib.LKLAttnProblem(**d)


def rows(**kw):
    d = dict(B=2, T=10, V=1000, sb=10000, st=1000, dtype=1)
    d.update(kw)
    return _lib.LKLLogits(**d)


def fwd(p, q=FAKE, strides=None, mask=None, lse=FAKE, ws=None, n=0):
    return _lib.lib().lkl_attn_forward(q, FAKE, FAKE, strides, mask, ctypes.byref(p), FAKE2, lse, ws,
                                       n, None)


def test_tensors_must_be_on_cuda():
    q = torch.randn(1, 2, 8, 16).half()
    for f in (attn, attn_forward):
        with pytest.raises(AssertionError, match="CUDA"):
            f(q, q, q)
    with pytest.raises(AssertionError, match="torch.Tensor"):
        attn(q.numpy(), q, q)
    x = torch.randn(2, 3, 50)
    with pytest.raises(AssertionError, match="CUDA"):
        token_logprobs(x, torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(AssertionError, match="CUDA"):
        logits_kl_align(x, x)


@pytest.mark.parametrize("kw,code", [
    (dict(Hq=6, Hkv=4), 2), (dict(Hq=0), 2), (dict(Hkv=0), 2), (dict(B=-1), 2), (dict(T=-1), 2),
    (dict(D=96), 3), (dict(D=512), 3), (dict(dtype=2), 4), (dict(dtype=7), 4),
    (dict(mask_dtype=9), 4), (dict(B=1 << 20, Hq=1 << 12, Hkv=1 << 12), 11)])
def test_attention_refuses_bad_problems(kw, code):
    p = prob(**kw)
    assert fwd(p) == code
    assert _lib.lib().lkl_attn_backward(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None,
                                        ctypes.byref(p), FAKE4, FAKE2, FAKE3, FAKE, 1 << 40,
                                        None) == code
    assert _lib.lib().lkl_attn_forward_workspace_size(ctypes.byref(p), 1) == 0
    assert _lib.lib().lkl_attn_backward_workspace_size(ctypes.byref(p), 1) == 0


def test_attention_refuses_bad_pointers_strides_and_scratch():
    p, L = prob(), _lib.lib()
    assert fwd(p, q=None) == 1
    assert fwd(p, q=ctypes.c_void_p(0x10001)) == 5
    assert fwd(p, lse=ctypes.c_void_p(0x10002)) == 5
    assert fwd(p, mask=ctypes.c_void_p(0x10004), ws=FAKE, n=1 << 20) == 5     # int64 mask
    n = L.lkl_attn_forward_workspace_size(ctypes.byref(p), 1)
    assert n == 256 * ((2 * 10 * 4 + 255) // 256)
    assert L.lkl_attn_forward_workspace_size(ctypes.byref(p), 0) == 0
    assert fwd(p, mask=FAKE, ws=FAKE, n=n - 1) == 6
    assert fwd(p, mask=FAKE, ws=None, n=n) == 6
    good = _lib.LKLStrides(b=300 * 512, h=128, t=512)
    for bad, at in ((_lib.LKLStrides(b=-8, h=128, t=512), 0), (_lib.LKLStrides(b=8, h=128, t=0), 3)):
        s = [good] * 4
        s[at] = bad
        assert fwd(p, strides=(_lib.LKLStrides * 4)(*s)) == 2
    need = L.lkl_attn_backward_workspace_size(ctypes.byref(p), 1)
    assert need % 256 == 0 and need >= n + 2 * 4 * 300 * 8

    def bwd(dk=FAKE2, ws=FAKE, n=256, strides=None):
        return L.lkl_attn_backward(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, strides, None,
                                   ctypes.byref(p), FAKE4, dk, FAKE3, ws, n, None)
    assert bwd() == 6
    assert bwd(dk=None) == 1
    for other in (FAKE, FAKE3, FAKE4):      # an input, dv, dq
        assert bwd(dk=other, n=1 << 40) == 10
    assert L.lkl_attn_forward(FAKE, FAKE3, FAKE4, None, None, ctypes.byref(p), FAKE3, FAKE, None, 0,
                              None) == 10
    s = [good] * 8
    s[6] = _lib.LKLStrides(b=300 * 512, h=0, t=512)
    assert bwd(n=1 << 40, strides=(_lib.LKLStrides * 8)(*s)) == 2
    assert fwd(prob(T=0), q=None) == 0 and fwd(prob(B=0), q=None) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 4), (dict(V=0), 2), (dict(B=-1), 2), (dict(st=-1), 2), (dict(V=1 << 31), 11),
    (dict(B=1 << 16, T=1 << 16), 11)])
def test_logits_refuse_bad_rows(kw, code):
    L, r, ok = _lib.lib(), rows(**kw), rows()
    b, o = ctypes.byref(r), ctypes.byref(ok)
    assert L.lkl_token_logprobs(FAKE, b, FAKE, -100, 0, FAKE, FAKE, FAKE, None, None, None) == code
    assert L.lkl_token_logprobs_backward(FAKE, b, FAKE, -100, FAKE, FAKE, FAKE, FAKE, FAKE2,
                                         None) == code
    for x, y in ((b, o), (o, b)):
        assert L.lkl_logits_kl_forward(FAKE, x, FAKE, y, None, 0, 1.0, FAKE, FAKE, FAKE, FAKE,
                                       1 << 20, None) == code
        assert L.lkl_logits_kl_backward(FAKE, x, FAKE, y, None, 0, 1.0, FAKE, FAKE, None, FAKE2,
                                        None) == code


def test_logits_refuse_bad_arguments():
    L, r = _lib.lib(), rows()
    b = ctypes.byref(r)

    def token(x=FAKE, ids=FAKE, k=0, tv=FAKE, ti=FAKE, rr=b):
        return L.lkl_token_logprobs(x, rr, ids, -100, k, FAKE, FAKE, FAKE, tv, ti, None)
    assert token(k=33) == 2 and token(k=-1) == 2
    assert token(k=3, rr=ctypes.byref(rows(V=2))) == 2
    assert token(x=None) == 1 and token(ids=None) == 1 and token(k=1, tv=None) == 1
    assert token(x=ctypes.c_void_p(0x10001)) == 5 and token(ids=ctypes.c_void_p(0x10004)) == 5
    assert token(rr=ctypes.byref(rows(T=0)), x=None) == 0

    def kl(t=b, mask=None, mdt=0, tau=1.0, ws=FAKE, n=1 << 20, loss=FAKE):
        return L.lkl_logits_kl_forward(FAKE, b, FAKE, t, mask, mdt, tau, FAKE, FAKE, loss, ws, n,
                                       None)
    for kw in (dict(V=999), dict(T=9), dict(B=1)):
        assert kl(t=ctypes.byref(rows(**kw))) == 2
    assert kl(t=ctypes.byref(rows(dtype=0))) == 4
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-45):
        assert kl(tau=tau) == 2
    assert kl(mask=FAKE, mdt=5) == 4 and kl(loss=None) == 1
    assert kl(n=L.lkl_logits_kl_workspace_size(b) - 1) == 6 and kl(ws=None) == 6
    # a gradient does not overwrite the logits
    assert L.lkl_token_logprobs_backward(FAKE, b, FAKE, -100, FAKE, FAKE, FAKE, FAKE, FAKE,
                                         None) == 10
    for x, y in ((FAKE, FAKE2), (FAKE2, FAKE)):
        assert L.lkl_logits_kl_backward(x, b, y, b, None, 0, 1.0, FAKE, FAKE, None, FAKE, None) == 10


def test_backward_scratch_of_a_group_beyond_8_gib():
    """One kv head whose dS tiles exceed 8 GiB runs in chunks of key tiles: the
    scratch asked for is 8 GiB of tiles and the fp32 dq of its query heads."""
    L, p = _lib.lib(), prob(B=1, Hq=8, Hkv=1, T=40000)
    n_t = (40000 + 127) // 128
    need = L.lkl_attn_backward_workspace_size(ctypes.byref(p), 0)
    stats, acc = 8 * n_t * 1024, 8 * 40000 * 128 * 4
    assert 8 * n_t * (n_t + 1) // 2 * 32768 > 8 << 30
    assert need >= stats + acc + (8 << 30)
    assert need < stats + acc + (8 << 30) + (1 << 30)
