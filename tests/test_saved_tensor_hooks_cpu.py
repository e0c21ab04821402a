"""What the autograd functions hand to the kernels when a saved-tensor hook gives
their tensors back in another layout: followed on the CPU, with a stand-in for the
library that records its arguments."""
import ctypes

import pytest
import torch

from linearard_b200 import _lib
from linearard_b200.attention import recompute
from linearard_b200.logits import _common, kl, token


class Recorder:
    """Stand-in for the loaded library: keeps the arguments of every call, does nothing."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 256 if name.endswith("workspace_size") else 0
        return call


@pytest.fixture
def recorder(monkeypatch):
    import contextlib
    r = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    for m in (recompute, kl, token):
        monkeypatch.setattr(m, "on_device", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(m, "raw_stream", lambda device: 0)
    return r


def held(unpack):
    """Hooks that keep what was given out, so that addresses can be looked up."""
    out = []

    def un(t):
        out.append(unpack(t))
        return out[-1]
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, un), out


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def strange(t):
    """The same values with a last stride other than 1."""
    return torch.stack([t, t], -1)[..., 0] if t.ndim else t


UNPACK = {"as it was": lambda t: t, "dense": dense, "strange": strange}


def span(t, strides):
    """One past the last element that strides (b, h, t) of a [B, H, T, D] tensor reach."""
    return sum((n - 1) * s for n, s in zip(t.shape[:3], strides)) + t.shape[3]


@pytest.mark.parametrize("unpack", UNPACK)
@pytest.mark.parametrize("layout", ["bthd", "fused", "bhtd"])
@pytest.mark.parametrize("mask", [False, True])
def test_attention_backward_reads_what_the_hook_gave_back(recorder, unpack, layout, mask):
    B, Hq, Hkv, T, D = 2, 4, 2, 16, 8

    def heads(H):
        if layout == "bhtd":
            return torch.randn(B, H, T, D).half()
        x = torch.randn(B, T, H, (2 if layout == "fused" else 1) * D).half()[..., -D:]
        return x.transpose(1, 2)
    q, k, v = (heads(H).requires_grad_(True) for H in (Hq, Hkv, Hkv))
    m = torch.ones(B, T, dtype=torch.int64) if mask else None
    prob = recompute._problem(q, k, True, _lib.LKL_MASK_I64, None)
    hooks, given = held(UNPACK[unpack])
    with hooks:
        out = recompute.AttnFn.apply(q, k, v, m, prob)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    args = recorder.calls["lkl_attn_backward"]
    strides = [tuple(args[6][3 * i:3 * i + 3]) for i in range(8)]
    for i, shape in enumerate([(B, Hq, T, D), (B, Hkv, T, D), (B, Hkv, T, D), (B, Hq, T, D)]):
        at = [t for t in given if t.data_ptr() == args[i] and tuple(t.shape) == shape]
        if unpack == "strange":     # copied: the kernels need a last stride of 1
            assert not at and strides[i] == (shape[1] * T * D, T * D, D)
            continue
        assert strides[i] == at[0].stride()[:3], i
        assert 2 * span(at[0], strides[i]) <= (at[0].untyped_storage().nbytes()
                                               - 2 * at[0].storage_offset())
    # the mask and the row statistics are read as dense tensors
    if unpack != "strange":
        assert any(t.data_ptr() == args[4] and t.is_contiguous() for t in given)
        assert (args[7] is not None) == mask
    for g, t in zip(grads, (q, k, v)):
        assert g.shape == t.shape


def test_attention_backward_refuses_other_types_from_a_hook(recorder):
    q = torch.randn(1, 2, 4, 8).half().requires_grad_(True)
    prob = recompute._problem(q, q, True, _lib.LKL_MASK_U8, None)
    for bad in (lambda t: t.float() if t.dtype == torch.float16 else t,
                lambda t: t.half() if t.dtype == torch.float32 else t,
                lambda t: t[..., :4]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            out = recompute.AttnFn.apply(q, q, q, None, prob)
        with pytest.raises(AssertionError, match="saved"):
            torch.autograd.grad(out.sum(), q)
        assert "lkl_attn_backward" not in recorder.calls


def rows_end(r):
    """One past the last element that a row descriptor reaches."""
    return (r.B - 1) * r.sb + (r.T - 1) * r.st + r.V


def check_rows(args, at, given, shape):
    """The kernel's row descriptor is that of the tensor it is given."""
    r = args[at + 1]._obj
    mine = [t for t in given if t.data_ptr() == args[at] and tuple(t.shape) == shape]
    assert (r.B, r.T, r.V) == shape
    if mine and mine[0].stride(-1) == 1:
        t = mine[0]
        assert (r.sb, r.st) == t.stride()[:2]
        assert rows_end(r) * t.element_size() <= (t.untyped_storage().nbytes()
                                                  - t.storage_offset() * t.element_size())
    else:                        # copied: rows have to be dense
        assert not any(t.data_ptr() == args[at] for t in given)
        assert (r.sb, r.st) == (shape[1] * shape[2], shape[2])


@pytest.mark.parametrize("unpack", UNPACK)
@pytest.mark.parametrize("cut", ["shift", "vocab", "whole"])
def test_token_backward_reads_what_the_hook_gave_back(recorder, unpack, cut):
    x = torch.randn(2, 6, 7)
    x = {"shift": x[:, :-1], "vocab": x[..., 1:5], "whole": x}[cut].requires_grad_(True)
    ids = torch.zeros(x.shape[:2], dtype=torch.int64)
    hooks, given = held(UNPACK[unpack])
    with hooks:
        outs = token.TokenLogprobsFn.apply(x, _common.rows_of(x), ids, 0, -100)
    (d,) = torch.autograd.grad(outs[0].sum(), x)
    args = recorder.calls["lkl_token_logprobs_backward"]
    check_rows(args, 0, given, tuple(x.shape))
    assert d.shape == x.shape
    if unpack != "strange":
        for k in (2, 4, 5):          # targets, lse, entropy
            assert any(t.data_ptr() == args[k] and t.is_contiguous() for t in given)
        n = ids.numel()
        assert args[1]._obj.lse_low == args[4] + 4 * n
        assert any(t.data_ptr() == args[4] and t.numel() == 2 * n for t in given)


@pytest.mark.parametrize("unpack", UNPACK)
@pytest.mark.parametrize("cut", ["shift", "vocab", "whole"])
@pytest.mark.parametrize("mask", [False, True])
def test_kl_backward_reads_what_the_hook_gave_back(recorder, unpack, cut, mask):
    s, t = torch.randn(2, 2, 6, 7).unbind(0)
    s, t = ({"shift": x[:, :-1], "vocab": x[..., 1:5], "whole": x}[cut] for x in (s, t))
    s = s.requires_grad_(True)
    m = torch.ones(s.shape[:2], dtype=torch.int64) if mask else None
    hooks, given = held(UNPACK[unpack])
    with hooks:
        loss = kl.LogitsKLAlignFn.apply(s, t, m, _lib.LKL_MASK_I64, 1.0,
                                        (_common.rows_of(s), _common.rows_of(t)))
    (d,) = torch.autograd.grad(loss, s)
    args = recorder.calls["lkl_logits_kl_backward"]
    check_rows(args, 0, given, tuple(s.shape))
    check_rows(args, 2, given, tuple(t.shape))
    assert d.shape == s.shape and (args[4] is not None) == mask
    if unpack != "strange":
        n = s.shape[0] * s.shape[1]      # the two log-sum-exps, each with what it lacks
        assert any(z.data_ptr() == args[7] and z.is_contiguous() and z.numel() == 4 * n
                   for z in given)
        assert args[8] == args[7] + 8 * n
        assert args[1]._obj.lse_low == args[7] + 4 * n and args[3]._obj.lse_low == args[8] + 4 * n


def test_logits_backward_refuses_other_types_from_a_hook(recorder):
    x = torch.randn(2, 6, 8).requires_grad_(True)
    ids = torch.zeros(2, 6, dtype=torch.int64)
    hooks = torch.autograd.graph.saved_tensors_hooks
    for bad in (lambda t: t.half() if t.is_floating_point() else t, lambda t: t[..., :4],
                lambda t: t if t.is_floating_point() else t.int()):
        with hooks(lambda t: t, bad):
            lp = token.TokenLogprobsFn.apply(x, _common.rows_of(x), ids, 0, -100)[0]
            loss = kl.LogitsKLAlignFn.apply(x, x.detach(), ids, _lib.LKL_MASK_I64, 1.0,
                                            (_common.rows_of(x),) * 2)
        for y in (lp.sum(), loss):
            with pytest.raises(AssertionError, match="saved"):
                torch.autograd.grad(y, x)
    assert not any("backward" in name for name in recorder.calls)
