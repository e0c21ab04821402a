"""The attention and its recomputing backward on a B200 against a float64
formulation, at the sizes, layouts and masks where tiles end."""
import pytest
import torch

from gpu_util import check_device_status, force_generic
from linearard_b200.attention import attn, attn_backward, attn_forward
from operator_refs import AttnRef, assert_within

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def make(B, Hq, Hkv, T, D, dtype, layout="bthd", seed=0, scale=1.3):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(H, s):
        if layout == "bthd":
            return (torch.randn(B, T, H, D, device="cuda", generator=g) * s).to(DT[dtype]).transpose(1, 2)
        if layout == "fused":      # heads of one wider projection
            return (torch.randn(B, T, H, 2 * D, device="cuda", generator=g) * s).to(
                DT[dtype])[..., D:].transpose(1, 2)
        if layout == "odd":        # no stride that TMA can read
            return (torch.randn(B, H, T, D + 1, device="cuda", generator=g) * s).to(DT[dtype])[..., 1:]
        return (torch.randn(B, H, T, D, device="cuda", generator=g) * s).to(DT[dtype])
    return one(Hq, scale), one(Hkv, scale), one(Hkv, 1.0), one(Hq, 1.0)


def check(q, k, v, g, mask=None, causal=True, sm_scale=None, backward=True):
    ref = AttnRef(q, k, v, mask, causal, sm_scale, g if backward else None)
    out, lse = attn_forward(q, k, v, mask, causal, sm_scale)
    assert_within(lse, ref.lse, ref.lse_tol, "lse")
    assert_within(out, ref.out, ref.out_tol, "out")
    if backward:
        dq, dk, dv = attn_backward(g, q, k, v, out, lse, mask, causal, sm_scale)
        assert_within(dv, ref.dv, ref.dv_tol, "dv")
        assert_within(dk, ref.dk, ref.dk_tol, "dk")
        assert_within(dq, ref.dq, ref.dq_tol, "dq")
        assert dq.stride() == (q.stride() if q.shape[1] > 1 and q.shape[0] > 1
                               and q.is_contiguous() else dq.stride())
    torch.cuda.synchronize()
    check_device_status()


def right_pad(B, T, lens):
    m = torch.zeros(B, T, dtype=torch.int64, device="cuda")
    for b in range(B):
        m[b, :lens[b % len(lens)]] = 1
    return m


@pytest.mark.parametrize("T", [1, 2, 7, 64, 127, 128, 129, 255, 256, 257, 384, 640, 1030])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(T, causal):
    check(*make(2, 4, 2, T, 128, "bf16"), causal=causal)


@pytest.mark.parametrize("D", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_head_dims(D, dtype):
    check(*make(1, 2, 1, 300, D, dtype))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 2), (6, 6)])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_heads(Hq, Hkv, D):
    check(*make(2, Hq, Hkv, 333, D, "bf16", "bhtd"))


@pytest.mark.parametrize("layout", ["bhtd", "bthd", "fused", "odd"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_layouts(layout, D):
    check(*make(2, 4, 2, 200, D, "fp16", layout))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", ["right", "left", "holes", "one", "none"])
def test_masks(D, causal, kind):
    B, T = 3, 421
    q, k, v, g = make(B, 4, 2, T, D, "bf16")
    m = right_pad(B, T, [421, 130, 3])
    if kind == "left":
        m = m.flip(1)
    elif kind == "holes":
        m = (torch.arange(T, device="cuda")[None] * 7 + torch.arange(B, device="cuda")[:, None]) % 5 != 0
    elif kind == "one":
        m = torch.zeros(B, T, dtype=torch.uint8, device="cuda")
        m[:, 300] = 1
    elif kind == "none":      # a sequence without any token
        m[1] = 0
    check(q, k, v, g, m, causal)


@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_what_removed_tokens_hold_reaches_nothing(D, poison):
    B, T = 2, 390
    q, k, v, g = make(B, 2, 1, T, D, "bf16", "bhtd")
    m = right_pad(B, T, [390, 201]).bool()
    m[0, 5:40] = False
    want = attn_forward(q, k, v, m)
    grads = attn_backward(g, q, k, v, *want, m)
    bad = [t.clone() for t in (q, k, v, g)]
    for t in bad:
        t.masked_fill_(~m[:, None, :, None], poison)
    out, lse = attn_forward(*bad[:3], m)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    out2 = out.masked_fill(~m[:, None, :, None], poison)
    for a, b in zip(attn_backward(bad[3], *bad[:3], out2, lse, m), grads):
        assert torch.equal(a, b)
    check(*bad, mask=m)


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64])
def test_mask_types_and_cpu_masks(mask_dtype):
    q, k, v, g = make(2, 2, 2, 140, 64, "bf16")
    m = right_pad(2, 140, [140, 77]).to(mask_dtype)
    check(q, k, v, g, m)
    check(q, k, v, g, m.cpu())


@pytest.mark.parametrize("sm_scale", [1.0, 0.01])
def test_scale(sm_scale):
    check(*make(1, 2, 2, 260, 128, "bf16", scale=0.7), sm_scale=sm_scale)


def test_large_scores_keep_their_rows():
    """Rows whose maximum moves by hundreds between tiles."""
    q, k, v, g = make(1, 2, 2, 700, 128, "bf16")
    k = (k.float() * torch.linspace(0.1, 12, 700, device="cuda")[None, None, :, None]).bfloat16()
    check(q, k, v, g)
    check(q, k.flip(2), v, g, causal=False)


def test_autograd_matches_and_broadcast_inputs():
    q, k, v, g = make(2, 4, 2, 150, 64, "bf16")
    want = attn_forward(q, k, v)[0]
    grads = attn_backward(g, q, k, v, *attn_forward(q, k, v))
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    out = attn(*leaves)
    out.backward(g)
    assert torch.equal(out, want)
    for leaf, d in zip(leaves, grads):
        assert torch.equal(leaf.grad, d)
    # one kv tensor seen by the whole batch, and as keys and values at once
    one = k[:1].detach().clone().requires_grad_(True)
    many = one.expand(2, -1, -1, -1)
    out = attn(q, many, many)
    (d_one,) = torch.autograd.grad(out, one, g)
    kk = k[:1].expand(2, -1, -1, -1)
    o, z = attn_forward(q, kk.contiguous(), kk.contiguous())
    _, dk, dv = attn_backward(g, q, kk.contiguous(), kk.contiguous(), o, z)
    torch.testing.assert_close(d_one, (dk + dv).sum(0, keepdim=True), rtol=2 ** -6, atol=2 ** -6)
    # the gradient of a sum is one number seen everywhere
    leaves[0].grad = None
    attn(*leaves).sum().backward()
    want = attn_backward(torch.ones_like(g), q, k, v, *attn_forward(q, k, v))[0]
    assert torch.equal(leaves[0].grad, want)


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_against_differences(causal):
    """Central differences of sum(out w) in float64 of the formula, along random
    directions: the derivative's own error is O(step^2)."""
    q, k, v, w = make(1, 2, 1, 70, 16, "fp16", scale=0.8)
    out, lse = attn_forward(q, k, v, causal=causal)
    grads = attn_backward(w, q, k, v, out, lse, causal=causal)
    ref = AttnRef(q, k, v, None, causal, None, w)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, (name, d) in enumerate(zip("qkv", grads)):
        x = [q.double(), k.double(), v.double()]
        e = torch.randn(x[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5

        def f(t):
            y = list(x)
            y[i] = x[i] + t * e
            kk, vv = (z.repeat_interleave(2, 1) for z in y[1:])
            s = (y[0] @ kk.transpose(-1, -2)) * 16 ** -0.5
            if causal:
                s = s.masked_fill(torch.ones(70, 70, device="cuda").triu(1).bool(), -torch.inf)
            return ((s.softmax(-1) @ vv) * w.double()).sum()
        slope = ((f(h) - f(-h)) / (2 * h)).item()
        tol = ((getattr(ref, f"d{name}_tol") * e.abs()).sum() + 1e-6).item()
        assert abs((d.double() * e).sum().item() - slope) <= tol, name


def test_same_bits_every_time_and_on_the_other_path():
    q, k, v, g = make(2, 4, 2, 600, 128, "bf16")
    m = right_pad(2, 600, [600, 345])
    first = None
    for _ in range(3):
        out, lse = attn_forward(q, k, v, m)
        got = (out, lse, *attn_backward(g, q, k, v, out, lse, m))
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, got))
        first = got
    with force_generic():
        check(q, k, v, g, m)


def test_rows_behind_the_tensor_stay():
    """Outputs at the end of a larger buffer: nothing past them is written."""
    from linearard_b200 import _lib
    import ctypes
    B, H, T, D = 1, 2, 130, 64
    q, k, v, g = (t.contiguous() for t in make(B, H, H, T, D, "bf16", "bhtd"))
    n = q.numel()
    bufs = [torch.full((n + 512,), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    lse = torch.full((B * H * T + 64,), 7.0, device="cuda")
    p = _lib.LKLAttnProblem(B=B, Hq=H, Hkv=H, T=T, D=D, dtype=1, causal=1, mask_dtype=1, sm_scale=0.125)
    L = _lib.lib()
    vp = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    st = torch.cuda.current_stream().cuda_stream
    nb = L.lkl_attn_backward_workspace_size(ctypes.byref(p), 0)
    ws = torch.empty(nb + 256, dtype=torch.uint8, device="cuda").fill_(9)
    assert L.lkl_attn_forward(vp(q), vp(k), vp(v), None, None, ctypes.byref(p), vp(bufs[0]), vp(lse),
                              None, 0, ctypes.c_void_p(st)) == 0
    assert L.lkl_attn_backward(vp(q), vp(k), vp(v), vp(bufs[0]), vp(lse), vp(g), None, None,
                               ctypes.byref(p), vp(bufs[1]), vp(bufs[2]), vp(bufs[3]), vp(ws), nb,
                               ctypes.c_void_p(st)) == 0
    torch.cuda.synchronize()
    for b in bufs:
        assert (b[n:] == 7).all() and (b[:n] != 7).any()
    assert (lse[B * H * T:] == 7).all() and (ws[nb:] == 9).all()


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (4, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("mask", [False, True])
def test_chunks_of_the_backward(Hq, Hkv, causal, mask):
    """Less scratch than asked for: fewer kv heads a launch, then key tiles of one
    kv head with dq summed over launches.  dk and dv keep their bits; dq is summed in
    another order."""
    import ctypes

    from linearard_b200 import _lib
    from linearard_b200.attention import recompute as R
    B, T, D = 2, 700, 128
    q, k, v, g = make(B, Hq, Hkv, T, D, "bf16", "bhtd")
    m = right_pad(B, T, [700, 290]) if mask else None
    out, lse = attn_forward(q, k, v, m, causal)
    want = attn_backward(g, q, k, v, out, lse, m, causal)
    ref = AttnRef(q, k, v, m, causal, None, g)
    prob = R._problem(q, k, causal, _lib.LKL_MASK_I64, None)
    L = _lib.lib()
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    full = L.lkl_attn_backward_workspace_size(ctypes.byref(prob), int(mask))
    n_t, G = 6, Hq // Hkv
    tiles = n_t * (n_t + 1) // 2 if causal else n_t * n_t
    base = full - B * Hq * tiles * 32768
    acc = G * T * D * 4
    sizes = [full, base + 3 * G * tiles * 32768, base + G * tiles * 32768,
             base + acc + 4 * G * n_t * 32768, base + acc + 2 * G * n_t * 32768,
             base + acc + G * n_t * 32768]
    for n in sizes:
        ws = torch.full((n + 256,), 0xFF, dtype=torch.uint8, device="cuda")
        grads = [torch.empty_like(t) for t in (q, k, v)]
        st = L.lkl_attn_backward(*(t.data_ptr() for t in (q, k, v, out, lse, g)), None, at(m),
                                 ctypes.byref(prob), *(t.data_ptr() for t in grads), ws.data_ptr(), n,
                                 R.raw_stream(q.device))
        assert st == 0
        assert (ws[n:] == 0xFF).all()
        assert torch.equal(grads[1], want[1]) and torch.equal(grads[2], want[2])
        assert_within(grads[0], ref.dq, ref.dq_tol, "dq")
    assert L.lkl_attn_backward(*(t.data_ptr() for t in (q, k, v, out, lse, g)), None, at(m),
                               ctypes.byref(prob), *(t.data_ptr() for t in grads), ws.data_ptr(),
                               sizes[-1] - 256, R.raw_stream(q.device)) == 6
    check_device_status()


def test_captured_and_replayed():
    q, k, v, g = make(1, 4, 2, 300, 128, "bf16")
    m = right_pad(1, 300, [211])
    attn_backward(g, q, k, v, *attn_forward(q, k, v, m), m)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            out, lse = attn_forward(q, k, v, m)
            grads = attn_backward(g, q, k, v, out, lse, m)
    for seed in (3, 4):
        for t, n in zip((q, k, v, g), make(1, 4, 2, 300, 128, "bf16", seed=seed)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = attn_forward(q, k, v, m)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        for a, b in zip(grads, attn_backward(g, q, k, v, *want, m)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    sets = [make(1, 4, 4, 900, 128, "bf16", seed=s) for s in (1, 2)]
    want = [attn_backward(g, q, k, v, *attn_forward(q, k, v)) for q, k, v, g in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, (q, k, v, g) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i] = attn_backward(g, q, k, v, *attn_forward(q, k, v))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_nothing_to_do():
    for B, T in ((0, 5), (2, 0)):
        q = torch.empty(B, 2, T, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = attn(q, q, q)
        assert out.shape == q.shape
        out.sum().backward()
        assert q.grad.shape == q.shape


@pytest.mark.parametrize("Hq,Hkv,causal,mask", [(2, 1, True, False), (1, 1, False, True),
                                                (4, 2, True, True)])
def test_long_key_tiles_are_shared(Hq, Hkv, causal, mask):
    """Few key tiles with many query tiles each: several blocks share one and their
    sums are joined.  The same bounds, and the same bits every time."""
    T = 4300
    q, k, v, g = make(1, Hq, Hkv, T, 64, "bf16")
    m = right_pad(1, T, [4111]) if mask else None
    check(q, k, v, g, m, causal)
    out, lse = attn_forward(q, k, v, m, causal)
    a, b = (attn_backward(g, q, k, v, out, lse, m, causal) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_through_autograd():
    """Forward and torch.autograd.grad inside one capture, after a warm-up on the
    capture's stream whose graph is gone (autograd ties the leaves of a living graph
    to the stream that it was built on)."""
    q, k, v, g = (t.detach() for t in make(1, 2, 2, 260, 64, "bf16"))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        torch.autograd.grad(attn(*leaves), leaves, g)
        with torch.cuda.graph(graph, stream=s):
            out = attn(*leaves)
            grads = torch.autograd.grad(out, leaves, g)
    graph.replay()
    torch.cuda.synchronize()
    o, z = attn_forward(q, k, v)
    assert torch.equal(out, o)
    for a, b in zip(grads, attn_backward(g, q, k, v, o, z)):
        assert torch.equal(a, b)


def test_no_second_derivative():
    q, k, v, g = make(1, 2, 2, 40, 64, "bf16")
    q = q.detach().requires_grad_(True)
    (d,) = torch.autograd.grad(attn(q, k, v), q, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), q)


def test_refusals():
    q, k, v, g = make(2, 4, 2, 40, 64, "bf16", "bhtd")
    for bad in ((q.float(), k, v), (q, k, v.half()), (q[..., :60], k[..., :60], v[..., :60]),
                (q[:, :3], k, v), (q, k[:, :, :30], v[:, :, :30]), (q, k, v[:, :1]),
                (q.transpose(2, 3), k, v), (q[0], k[0], v[0])):
        with pytest.raises(AssertionError):
            attn(*bad)
    for mask in (torch.ones(2, 41, device="cuda", dtype=torch.int64), torch.ones(2, 40, device="cuda"),
                 torch.ones(2, 1, 40, 40, device="cuda", dtype=torch.bool), [1, 2]):
        with pytest.raises(AssertionError):
            attn(q, k, v, mask)
    for sc in (0.0, -1.0, float("nan"), float("inf"), "1"):
        with pytest.raises(AssertionError):
            attn(q, k, v, sm_scale=sc)
    out, lse = attn_forward(q, k, v)
    for bad in ((g.float(), out, lse), (g, out[:, :2], lse), (g, out, lse.half()), (g, out, lse[:, :2])):
        with pytest.raises(AssertionError):
            attn_backward(bad[0], q, k, v, *bad[1:])


@pytest.mark.parametrize("D", [16, 128, 256])
@pytest.mark.parametrize("T", [2, 3, 5, 8, 33, 128])
def test_short_sequences_keep_small_gradients(T, D):
    """Where one key has most of a row, dS is a small difference of dout . v and
    delta: short sequences take delta from the probabilities, so that what is left are
    the roundings of dS and of the results, u each and relative to their size."""
    q, k, v, g = make(2, 4, 4, T, D, "bf16", seed=T, scale=2.2)
    ref = AttnRef(q, k, v, None, True, None, g)
    out, lse = attn_forward(q, k, v)
    dq, dk, _ = attn_backward(g, q, k, v, out, lse)
    u = 2.0 ** -8
    kk, qq, gg, vv = (t.double() for t in (k, q, g, v))
    S = (qq @ kk.transpose(-1, -2)) * D ** -0.5
    keep = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    P = S.masked_fill(~keep, -torch.inf).softmax(-1)
    dP = gg @ vv.transpose(-1, -2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    # fp32: the sums behind S, dP and delta, on terms of size P |dout||v|
    c = (2 * D + 64) * 2.0 ** -24
    mag = gg.abs() @ vv.abs().transpose(-1, -2)
    size = (qq.abs() @ kk.abs().transpose(-1, -2)) * D ** -0.5
    top = torch.where(keep, size, 0.0).amax(-1, keepdim=True)
    tol = torch.where(keep, u * dS.abs() + P * (mag + (P * mag).sum(-1, keepdim=True))
                      * (c * (2 + 2 * top) + 2.0 ** -18), 0.0) + 2.0 ** -126
    assert_within(dq, ref.dq, D ** -0.5 * tol @ kk.abs() * (1 + u) + u * ref.dq.abs() + 1e-30, "dq")
    assert_within(dk, ref.dk, D ** -0.5 * tol.transpose(-1, -2) @ qq.abs() * (1 + u)
                  + u * ref.dk.abs() + 1e-30, "dk")


@pytest.mark.parametrize("causal, T, D", [
    (True, 129, 16), (True, 256, 128), (True, 300, 64), (True, 300, 256), (True, 1000, 128),
    (False, 200, 32), (False, 256, 128),
])
def test_rows_of_few_keys_keep_small_gradients(causal, T, D):
    """Rows that see at most 256 keys take delta from the probabilities in a sequence of any
    length, so that their dq holds no more than the roundings of dS and of the result."""
    n, H, Hkv = min(T, 256), 4, 2
    q, k, v, g = make(2, H, Hkv, T, D, "bf16", seed=T, scale=2.2)
    out, lse = attn_forward(q, k, v, causal=causal)
    dq, _, _ = attn_backward(g, q, k, v, out, lse, causal=causal)
    qq, gg = q[:, :, :n].double(), g[:, :, :n].double()
    kk, vv = (t[:, :, :n].double().repeat_interleave(H // Hkv, 1) for t in (k, v))
    S = (qq @ kk.transpose(-1, -2)) * D ** -0.5
    keep = torch.ones(n, n, dtype=torch.bool, device="cuda")
    keep = keep.tril() if causal else keep
    P = S.masked_fill(~keep, -torch.inf).softmax(-1)
    dP = gg @ vv.transpose(-1, -2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    # fp32 as above; a sum over up to 256 keys instead of 128 behind dq and delta
    u, c = 2.0 ** -8, (2 * D + 512) * 2.0 ** -24
    mag = gg.abs() @ vv.abs().transpose(-1, -2)
    size = (qq.abs() @ kk.abs().transpose(-1, -2)) * D ** -0.5
    top = torch.where(keep, size, 0.0).amax(-1, keepdim=True)
    tol = torch.where(keep, u * dS.abs() + P * (mag + (P * mag).sum(-1, keepdim=True))
                      * (c * (2 + 2 * top) + 2.0 ** -18), 0.0) + 2.0 ** -126
    exact = D ** -0.5 * dS @ kk
    assert_within(dq[:, :, :n], exact, D ** -0.5 * tol @ kk.abs() * (1 + u) + u * exact.abs()
                  + 1e-30, "dq")
