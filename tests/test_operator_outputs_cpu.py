"""What the logits operators return: tensors of their own, which a user may change in
place.  On the CPU, with a stand-in for the library."""
import contextlib

import pytest
import torch

from linearard_b200 import _lib
from linearard_b200.logits import _common, kl, token


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    class Library:
        def __getattr__(self, name):
            return lambda *a: 256 if name.endswith("workspace_size") else 0
    monkeypatch.setattr(_lib, "lib", Library)
    for m in (token, kl):
        monkeypatch.setattr(m, "on_device", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(m, "raw_stream", lambda device: 0)


def token_outputs(x):
    ids = torch.zeros(x.shape[:-1], dtype=torch.int64)
    return token.TokenLogprobsFn.apply(x, _common.rows_of(x), ids, 0, -100)[:2]


def test_token_outputs_may_be_changed_in_place():
    x = torch.randn(2, 3, 5, requires_grad=True)
    logprob, entropy = token_outputs(x)
    logprob.mul_(2.0)
    logprob.masked_fill_(torch.ones(2, 3, dtype=torch.bool), 0.0)
    torch.autograd.grad(logprob.sum() + entropy.sum(), x)
    logprob, entropy = token_outputs(x)
    with torch.no_grad():
        logprob.zero_()
    torch.autograd.grad((logprob + entropy).sum(), x)


def test_outputs_share_no_storage():
    x = torch.randn(2, 3, 5)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    outs = list(token._forward(x, _common.rows_of(x), ids, 2, -100))
    rows = _common.rows_of(x)
    outs += kl._forward(x, x, None, _lib.LKL_MASK_U8, 1.0, (rows, rows))
    assert len({t.untyped_storage().data_ptr() for t in outs}) == len(outs)
    assert not any(t._is_view() for t in outs)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor does not require grad, and its tangent would be lost."""
    import torch.autograd.forward_ad as fwad
    monkeypatch.setattr(token, "check_logits", lambda x: None)
    x, ids = torch.randn(3, 5), torch.zeros(3, dtype=torch.int64)
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            token.token_logprobs(fwad.make_dual(x, torch.ones_like(x)), ids)
        token.token_logprobs(x, ids)
    token.token_logprobs(x, ids)


def test_ignore_index_beyond_64_bits_is_refused(monkeypatch):
    """It would wrap into another number on its way to the kernel: 2^64 - 100 into -100."""
    monkeypatch.setattr(token, "check_logits", lambda x: None)
    x, ids = torch.randn(3, 5), torch.zeros(3, dtype=torch.int64)
    for n in (2 ** 64 - 100, 2 ** 63, -2 ** 63 - 1):
        with pytest.raises(AssertionError, match="ignore_index"):
            token.token_logprobs(x, ids, ignore_index=n)
    for n in (2 ** 63 - 1, -2 ** 63, 0):
        token.token_logprobs(x, ids, ignore_index=n)
