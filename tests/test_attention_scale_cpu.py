"""Scales that single precision does not hold are refused, from Python and from C."""
import ctypes

import pytest
import torch

from linearard_b200 import _lib
from linearard_b200.attention import recompute


@pytest.mark.parametrize("sc", [1e-46, 1e-39, 2e38, 1e39, float("nan"), float("inf")])
def test_scale_out_of_range(sc):
    q = torch.empty(1, 2, 8, 16).half()
    with pytest.raises(AssertionError, match="sm_scale"):
        recompute._problem(q, q, True, 1, sc)
    p = _lib.LKLAttnProblem(B=1, Hq=2, Hkv=2, T=8, D=16, dtype=0, causal=1, mask_dtype=1,
                            sm_scale=sc)
    if p.sm_scale == 0.0:       # what C sees of 1e-46 asks for the default
        return
    x, y = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x20000)
    L = _lib.lib()
    assert L.lkl_attn_forward(x, x, x, None, None, ctypes.byref(p), y, x, None, 0, None) == 2
    assert L.lkl_attn_backward(x, x, x, x, x, x, None, None, ctypes.byref(p), y, y, y, x, 1 << 30,
                               None) == 2


def test_scales_of_the_whole_range_are_taken():
    q = torch.empty(1, 2, 8, 16).half()
    for sc in (2.0 ** -126, 1e-30, 1, 1e38):
        assert recompute._problem(q, q, True, 1, sc).sm_scale == pytest.approx(sc, rel=1e-6)


def test_few_elements_ask_for_no_tile_scratch():
    """Heads of at most 512 elements never reach the kernels that hand over tiles: row
    statistics alone, 1 KB a head."""
    L = _lib.lib()

    def need(**kw):
        p = _lib.LKLAttnProblem(**{**dict(B=4, Hq=64, Hkv=64, T=8, D=64, dtype=1, causal=1,
                                          mask_dtype=1, sm_scale=0.0), **kw})
        return L.lkl_attn_backward_workspace_size(ctypes.byref(p), 0)
    for T, D in ((8, 64), (4, 128), (64, 8)):
        assert need(T=T, D=D) == 4 * 64 * 1024
    assert need(T=9) >= 4 * 64 * (1024 + 32768)
