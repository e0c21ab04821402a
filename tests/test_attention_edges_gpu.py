"""Attention calls at the edges of what its arguments allow: scales, masks that leave
few keys, memory orders, shared key tiles of every head dim."""
import pytest
import torch

from linearard_b200.attention import attn, attn_backward, attn_forward
from operator_refs import AttnRef, assert_within
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


def sees_few(m, causal):
    """[B, T] bool: kept rows that see at most 256 keys."""
    seen = m.cumsum(1) if causal else m.sum(1, keepdim=True).expand_as(m)
    return m & (seen <= 256)


@pytest.mark.parametrize("kind", ["left", "short", "holes", "right"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,D", [(300, 64), (700, 16), (700, 128), (1100, 256), (9000, 32)])
def test_rows_of_few_keys_under_a_mask(kind, causal, T, D):
    """What decides is how many keys a row sees, not where it stands: rows of at most 256
    keys take delta from the probabilities, so that their dq holds no more than the
    roundings of dS and of the result, and so does dk where every row is one of them."""
    B, H, Hkv = 3, 4, 2
    # scores of a few units: the bound on their fp32 sums stays below what a rounded out costs
    q, k, v, g = make(B, H, Hkv, T, D, "bf16", seed=T, scale=1.1)
    m = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    for b, n in enumerate((2, 200, T - 20)):
        if kind == "left":
            m[b, T - n:] = True
        elif kind == "holes":
            m[b, torch.randperm(T, device="cuda", generator=torch.Generator("cuda").manual_seed(b))[:n]] = True
        elif kind == "short":        # a short sequence behind a page of padding
            m[b, T // 3:T // 3 + min(n, 9 + 100 * b)] = True
        else:
            m[b, :n] = True
    out, lse = attn_forward(q, k, v, m, causal)
    dq, dk, _ = attn_backward(g, q, k, v, out, lse, m, causal)
    u = 2.0 ** -8
    few = sees_few(m, causal)
    for b in range(B):
        rows = few[b].nonzero()[:, 0]
        n = len(rows)
        if n == 0:
            continue
        qq, gg = q[b][:, rows].double(), g[b][:, rows].double()
        kk, vv = (t[b][:, rows].double().repeat_interleave(H // Hkv, 0) for t in (k, v))
        keep = torch.ones(n, n, dtype=torch.bool, device="cuda")
        keep = keep.tril() if causal else keep
        P = ((qq @ kk.transpose(-1, -2)) * D ** -0.5).masked_fill(~keep, -torch.inf).softmax(-1)
        dP = gg @ vv.transpose(-1, -2)
        dS = P * (dP - (P * dP).sum(-1, keepdim=True))
        # fp32: the sums of D products behind S (twice: for delta and for dS) and dP, of n
        # products behind delta and the results, on terms of size P |dout||v|
        c = (2 * D + 2 * n) * 2.0 ** -24
        mag = gg.abs() @ vv.abs().transpose(-1, -2)
        size = (qq.abs() @ kk.abs().transpose(-1, -2)) * D ** -0.5
        top = torch.where(keep, size, 0.0).amax(-1, keepdim=True)
        tol = torch.where(keep, u * dS.abs() + P * (mag + (P * mag).sum(-1, keepdim=True))
                          * (c * (2 + 2 * top) + 2.0 ** -18), 0.0) + 2.0 ** -126
        sc = D ** -0.5
        want = sc * dS @ kk
        assert_within(dq[b][:, rows], want, sc * tol @ kk.abs() * (1 + u) + u * want.abs() + 1e-30,
                      f"dq of sequence {b}")
        if n == int(m[b].sum()):
            def heads(x):
                return x.view(Hkv, H // Hkv, n, D).sum(1)
            want = heads(sc * dS.transpose(-1, -2) @ qq)
            tol = heads(sc * tol.transpose(-1, -2) @ qq.abs()) * (1 + u) + u * want.abs() + 1e-30
            assert_within(dk[b][:, rows], want, tol, f"dk of sequence {b}")
    if T < 9000:                 # the whole result, in [T, T] maps of 64 bits
        check(q, k, v, g, m, causal)


@pytest.mark.parametrize("layout", ["bhtd", "bthd", "fused", "odd"])
@pytest.mark.parametrize("D", [64, 256])
def test_results_follow_the_memory_order_of_their_tensors(layout, D):
    """out in the order of heads and tokens of q; dq, dk and dv in that of q, k and v."""
    B, Hq, Hkv, T = 2, 4, 2, 150
    q, k, v, g = make(B, Hq, Hkv, T, D, "bf16", layout)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    auto = attn(*leaves)
    out, lse = attn_forward(q, k, v)

    def order(H):
        return (T * H * D, D, H * D, 1) if layout in ("bthd", "fused") else (H * T * D, T * D, D, 1)
    assert out.stride() == auto.stride() == order(Hq)
    for d, H in zip(attn_backward(g, q, k, v, out, lse), (Hq, Hkv, Hkv)):
        assert d.stride() == order(H)
    for d, H in zip(torch.autograd.grad(auto, leaves, g), (Hq, Hkv, Hkv)):
        assert d.stride() == order(H)
    # tensors of different orders at once: each keeps its own
    mixed = attn_backward(g, q, k.contiguous(), v, out, lse)
    assert mixed[0].stride() == order(Hq) and mixed[2].stride() == order(Hkv)
    assert mixed[1].is_contiguous()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,D", [(1, 128), (4, 128), (2, 64), (8, 64), (7, 32), (16, 32), (8, 16),
                                 (32, 16), (64, 8)])
@pytest.mark.parametrize("mask", [False, True])
def test_sequences_of_few_elements_carry_their_results_rounding_alone(dtype, causal, T, D, mask):
    """Up to 512 elements a head everything before the results is fp32: the bounds are those
    of 32-bit inputs and half a step of each result."""
    q, k, v, g = make(3, 4, 2, T, D, dtype, seed=T + D)
    m = right_pad(3, T, [T, max(1, T // 2), max(1, T - 1)]) if mask else None
    ref = AttnRef(*(t.float() for t in (q, k, v)), m, causal, None, g.float())
    out, lse = attn_forward(q, k, v, m, causal)
    grads = attn_backward(g, q, k, v, out, lse, m, causal)
    u, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == "fp16" else (2.0 ** -8, 2.0 ** -133)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        want = getattr(ref, name)
        tol = getattr(ref, name + "_tol") * (1 + u) + u * want.abs() + tiny
        assert_within(got, want, tol, name)
    assert_within(lse, ref.lse, ref.lse_tol, "lse")
