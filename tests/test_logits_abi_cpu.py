"""The row descriptors' second part of the log-sum-exp through the C ABI: refusals."""
import ctypes

from linearard_b200 import _lib

FAKE = [ctypes.c_void_p(0x10000 * i) for i in range(1, 8)]


def rows(low=0):
    return _lib.LKLLogits(B=2, T=10, V=1000, sb=10000, st=1000, dtype=1, lse_low=low)


def kl(s, t, lse_s=FAKE[3], lse_t=FAKE[4]):
    L, x, y = _lib.lib(), ctypes.byref(s), ctypes.byref(t)
    fwd = L.lkl_logits_kl_forward(FAKE[0], x, FAKE[1], y, None, 0, 1.0, lse_s, lse_t, FAKE[5],
                                  FAKE[6], 1 << 20, None)
    return fwd, L.lkl_logits_kl_backward(FAKE[0], x, FAKE[1], y, None, 0, 1.0, lse_s, lse_t, None,
                                         FAKE[2], None)


def token(r):
    L, b = _lib.lib(), ctypes.byref(r)
    fwd = L.lkl_token_logprobs(FAKE[0], b, FAKE[1], -100, 0, FAKE[2], FAKE[3], FAKE[4], None, None,
                               None)
    return fwd, L.lkl_token_logprobs_backward(FAKE[0], b, FAKE[1], -100, FAKE[4], FAKE[3], None,
                                              None, FAKE[2], None)


def test_low_parts_are_arrays_of_their_own():
    low = 0x900000
    assert kl(rows(low), rows(low)) == (10, 10)            # one for both models
    for at in (FAKE[3].value, FAKE[4].value):              # a log-sum-exp itself
        assert kl(rows(at), rows()) == (10, 10) and kl(rows(), rows(at)) == (10, 10)
    assert token(rows(FAKE[4].value)) == (10, 10)
    assert kl(rows(low + 2), rows()) == (5, 5) and token(rows(low + 2)) == (5, 5)


def test_descriptors_without_one_are_taken():
    """Past every check the call looks for the device of the logits, which is none here."""
    r = rows()
    assert kl(r, r) == (8, 8) and token(r) == (8, 8)
    assert kl(rows(0x900000), rows(0xA00000)) == (8, 8)
