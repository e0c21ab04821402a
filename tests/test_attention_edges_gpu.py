"""Attention calls at the edges of what its arguments allow: scales, masks that leave
few keys, memory orders, shared key tiles of every head dim."""
import pytest
import torch

from test_attention_gpu import check, make, right_pad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sm_scale", [1e-28, 1e-30, 1e-37, 2.0 ** -126])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_small_scales_keep_removed_keys_out(sm_scale, causal, D):
    """A removed key has no weight however small the scale makes the scores."""
    q, k, v, g = make(2, 2, 1, 300, D, "bf16")
    check(q, k, v, g, right_pad(2, 300, [300, 70]).flip(1), causal, sm_scale, backward=False)
    check(q, k, v, g, None, causal, sm_scale, backward=False)
    if sm_scale > 1e-35:        # below, dq and dk are subnormal
        check(q, k, v, g, right_pad(2, 300, [300, 70]), causal, sm_scale)


@pytest.mark.parametrize("D", [8, 32, 128])
@pytest.mark.parametrize("Hq,Hkv,causal,mask", [(2, 1, True, False), (1, 1, False, True),
                                                (4, 2, True, True)])
def test_shared_key_tiles_of_every_head_dim(D, Hq, Hkv, causal, mask):
    """Few long key tiles, each the work of several blocks, whose sums have D columns; the
    last tile ends inside a warp."""
    q, k, v, g = make(1, Hq, Hkv, 4300, D, "bf16")
    check(q, k, v, g, right_pad(1, 4300, [4111]) if mask else None, causal)
