"""The logits operators on a B200 against float64: odd vocabularies, views,
-inf logits, ties, masks, and their gradients."""
import pytest
import torch

from linearard_b200.logits import (logits_kl_align, logits_kl_backward, logits_kl_forward,
                                   token_logprobs)
from operator_refs import KLRef, TokenRef, assert_within, row_tol

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def logits(*shape, dtype="bf16", seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(DT[dtype])


def check_token(x, ids, top_k=0, ignore=-100, g=None, h=None):
    ref = TokenRef(x, ids, top_k, ignore, g, h)
    leaf = x.detach().requires_grad_(True)
    r = token_logprobs(leaf, ids, top_k, ignore)
    assert_within(r.logprob, ref.logprob, ref.logprob_tol, "logprob")
    assert_within(r.entropy, ref.entropy, ref.entropy_tol, "entropy")
    if top_k:
        assert torch.equal(r.top_indices, ref.top_indices)
        lp = torch.where(ref.top_logprobs == -torch.inf, 0.0, ref.top_logprobs)
        got = torch.where(ref.top_logprobs == -torch.inf,
                          torch.where(r.top_logprobs == -torch.inf, 0.0, torch.nan),
                          r.top_logprobs.double())
        assert_within(got, lp, ref.logprob_tol[..., None].expand_as(lp), "top_logprobs")
    else:
        assert r.top_logprobs is None and r.top_indices is None
    if g is not None or h is not None:
        outs = [(o, d) for o, d in ((r.logprob, g), (r.entropy, h)) if d is not None]
        (d,) = torch.autograd.grad([o for o, _ in outs], leaf, [d for _, d in outs])
        assert d.dtype == x.dtype and d.is_contiguous()
        assert_within(d, ref.d, ref.d_tol, "d_logits")


@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 255, 1000, 4099, 32000, 50257, 131075])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_token_vocabularies(V, dtype):
    B, T = 2, 5
    x = logits(B, T, V, dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, V, (B, T), device="cuda", generator=gen)
    ids[0, 2] = -100
    g, h = torch.randn(2, B, T, device="cuda", generator=gen).unbind(0)
    check_token(x, ids, min(V, 20), g=g, h=h)


@pytest.mark.parametrize("rows", [1, 3, 40, 147, 149, 700, 2500])
def test_token_row_counts(rows):
    x = logits(rows, 9000, dtype="bf16")
    ids = torch.arange(rows, device="cuda") * 3 % 9000
    check_token(x, ids, 5, g=torch.ones(rows, device="cuda"))


@pytest.mark.parametrize("top_k", [0, 1, 2, 31, 32])
@pytest.mark.parametrize("order", ["up", "down", "equal", "steps"])
def test_token_top_k_orders_and_ties(top_k, order):
    V = 20011
    i = torch.arange(V, device="cuda", dtype=torch.float32)
    row = {"up": i / 1000, "down": -i / 1000, "equal": i * 0 + 1.5, "steps": (i % 97) / 8}[order]
    x = torch.stack([row, row.flip(0), row.roll(777)]).to(torch.float32)
    check_token(x, torch.tensor([0, 5, V - 1], device="cuda"), top_k)
    check_token(x.bfloat16(), torch.tensor([0, 5, V - 1], device="cuda"), top_k)


@pytest.mark.parametrize("cut", ["shift", "vocab", "both", "offset"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_token_views(cut, dtype):
    big = logits(3, 12, 5003, dtype=dtype)
    x = {"shift": big[:, :-1], "vocab": big[..., :4001], "both": big[:, 1:, 2:4999],
         "offset": big[1:, :, 1:]}[cut]
    ids = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(2))
    g = torch.randn(x.shape[:-1], device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    check_token(x, ids, 3, g=g, h=g * 0.3)
    check_token(x[0], ids[0], 3, g=g[0])


def test_token_minus_infinity():
    x = logits(4, 3000, dtype="fp32")
    x[0, 100:] = -torch.inf
    x[1, ::2] = -torch.inf
    x[2] = -torch.inf
    x[2, 77] = 3.0                       # certain
    x[3, 0] = torch.finfo(torch.float32).min
    ids = torch.tensor([3, 5, 77, 0], device="cuda")
    check_token(x[[0, 1, 2]], ids[[0, 1, 2]], 32, g=torch.ones(3, device="cuda"),
                h=torch.ones(3, device="cuda"))
    r = token_logprobs(x[3:], ids[3:], 4)
    assert r.logprob.item() == pytest.approx(torch.finfo(torch.float32).min, rel=1e-6)
    assert torch.isfinite(r.entropy).all()
    # a target without probability
    r = token_logprobs(x[:1], torch.tensor([200], device="cuda"))
    assert r.logprob.item() == -torch.inf


def test_token_not_a_number():
    x = logits(5, 3000, dtype="bf16")
    x[0, 17] = torch.nan
    x[1, 2900] = torch.inf
    x[2] = -torch.inf
    ids = torch.tensor([1, 1, 1, 3000, -7], device="cuda")
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, ids, 3)
    assert r.logprob.isnan().all()
    assert r.entropy[:3].isnan().all() and torch.isfinite(r.entropy[3:]).all()
    assert ((r.top_indices >= 0) & (r.top_indices < 3000)).all()
    (d,) = torch.autograd.grad(r.logprob, leaf, torch.ones(5, device="cuda"))
    assert d.isnan().all(dim=1).all()


def test_token_ignore_index():
    x = logits(2, 6, 999, dtype="bf16")
    ids = torch.full((2, 6), 998, device="cuda")
    ids[1] = 0
    check_token(x, ids, 2, ignore=0, g=torch.ones(2, 6, device="cuda"))
    leaf = x.detach().requires_grad_(True)
    r = token_logprobs(leaf, ids, ignore_index=0)
    (d,) = torch.autograd.grad(r.logprob.sum(), leaf)
    assert (r.logprob[1] == 0).all() and (d[1] == 0).all() and (d[0] != 0).any()


def test_token_strided_targets_and_gradients():
    x = logits(3, 7, 511, dtype="fp32")
    ids = torch.randint(0, 511, (7, 3), device="cuda").t()
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, ids)
    r.logprob.sum().backward()           # the gradient is one number seen everywhere
    want = TokenRef(x, ids, g=torch.ones(3, 7, device="cuda"))
    assert_within(leaf.grad, want.d, want.d_tol, "d_logits")


def test_token_gradient_against_differences():
    x = logits(3, 200, dtype="fp32")
    ids = torch.tensor([0, 150, -100], device="cuda")
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, ids)
    wl, we = torch.tensor([1.0, -2.0, 3.0], device="cuda"), torch.tensor([0.5, 1.0, -1.0], device="cuda")
    (d,) = torch.autograd.grad((r.logprob * wl).sum() + (r.entropy * we).sum(), leaf)
    gen = torch.Generator(device="cuda").manual_seed(5)
    e = torch.randn(x.shape, device="cuda", dtype=torch.float64, generator=gen)
    ref = TokenRef(x, ids, g=wl, h=we)

    def f(t):
        q = TokenRef(x.double() + t * e, ids)
        return ((q.logprob * wl).sum() + (q.entropy * we).sum()).item()
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs((d.double() * e).sum().item() - slope) <= (ref.d_tol * e.abs()).sum().item() + 1e-6


def check_kl(s, t, mask=None, tau=1.0):
    ref = KLRef(s, t, mask, tau)
    leaf = s.detach().requires_grad_(True)
    loss = logits_kl_align(leaf, t, mask, tau)
    assert loss.shape == () and loss.dtype == torch.float32
    assert_within(loss, ref.loss, ref.loss_tol, "loss")
    (d,) = torch.autograd.grad(loss, leaf)
    assert d.dtype == s.dtype and d.is_contiguous()
    assert_within(d, ref.d, ref.d_tol, "ds")
    got, lse_s, lse_t = logits_kl_forward(s, t, mask, tau)
    assert torch.equal(got, loss.detach())
    V = s.shape[-1]
    assert_within(lse_s, ref.lse_s, row_tol(s.double() / tau, V) + 1e-7, "lse_s")
    assert_within(lse_t, ref.lse_t, row_tol(t.double() / tau, V) + 1e-7, "lse_t")
    two = logits_kl_backward(s, t, lse_s, lse_t, mask, tau, torch.tensor(-2.0, device="cuda"))
    # -2 d itself is rounded elsewhere where d is subnormal
    assert_within(two, -2 * ref.d, 2 * ref.d_tol, "dloss = -2")


@pytest.mark.parametrize("V", [1, 2, 9, 63, 1000, 4099, 32000, 50257])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_kl_vocabularies(V, dtype):
    t = logits(2, 5, V, dtype=dtype)
    s = (t.float() + logits(2, 5, V, dtype="fp32", seed=1, scale=0.5)).to(DT[dtype])
    check_kl(s, t)


@pytest.mark.parametrize("rows", [1, 30, 149, 800, 3000])
def test_kl_row_counts(rows):
    check_kl(logits(rows, 5000, seed=1), logits(rows, 5000, seed=2))


@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0, 8.0])
@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64])
def test_kl_masks_and_temperatures(tau, mask_dtype):
    s, t = logits(3, 11, 777, seed=1), logits(3, 11, 777, seed=2)
    m = (torch.arange(33, device="cuda").view(3, 11) % 4 != 1).to(mask_dtype)
    m[1] = 0
    bad = m == 0
    s[bad], t[bad] = torch.nan, torch.inf
    ref_s, ref_t = (torch.where(bad[..., None], 0.0, x.float()).bfloat16() for x in (s, t))
    ref = KLRef(ref_s, ref_t, m, tau)
    leaf = s.requires_grad_(True)
    for mask in (m, m.cpu()):
        loss = logits_kl_align(leaf, t, mask, tau)
        (d,) = torch.autograd.grad(loss, leaf)
        assert_within(loss, ref.loss, ref.loss_tol, "loss")
        assert_within(d, ref.d, ref.d_tol, "ds")
        assert (d[bad] == 0).all()
    assert logits_kl_align(s, t, torch.zeros_like(m)).item() == 0


@pytest.mark.parametrize("cut", ["shift", "vocab", "mixed"])
def test_kl_views(cut):
    a, b = logits(3, 9, 2003, seed=1), logits(3, 9, 2003, seed=2)
    if cut == "shift":
        a, b = a[:, :-1], b[:, :-1]
    elif cut == "vocab":
        a, b = a[..., 3:1999], b[..., 3:1999]
    else:                # rows that start at different offsets from 16 bytes
        a, b = a[..., 1:2000], b[..., 4:].contiguous()
    check_kl(a, b, torch.ones(3, 10, device="cuda", dtype=torch.int64)[:, :a.shape[1]])
    check_kl(a[1], b[1])


def test_kl_minus_infinity():
    s, t = logits(3, 700, dtype="fp32", seed=1), logits(3, 700, dtype="fp32", seed=2)
    t[0, ::3] = -torch.inf               # a teacher that excludes tokens
    s[1, 5:9] = t[1, 5:9] = -torch.inf   # both exclude them
    check_kl(s[:2], t[:2])
    s[2, 4] = -torch.inf                 # the student excludes what the teacher gives
    loss = logits_kl_align(s.requires_grad_(True), t)
    assert loss.item() == torch.inf
    assert torch.isfinite(torch.autograd.grad(loss, s)[0]).all()


def test_kl_of_equal_logits_is_zero():
    x = logits(4, 5, 3001, dtype="bf16", scale=4.0)
    leaf = x.requires_grad_(True)
    loss = logits_kl_align(leaf, x.detach())
    assert loss.item() == 0.0
    assert (torch.autograd.grad(loss, leaf)[0] == 0).all()


def test_kl_gradient_against_differences():
    s, t = logits(3, 100, dtype="fp32", seed=1), logits(3, 100, dtype="fp32", seed=2)
    leaf = s.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(logits_kl_align(leaf, t, temperature=1.5) * 3, leaf)
    e = torch.randn(s.shape, device="cuda", dtype=torch.float64,
                    generator=torch.Generator(device="cuda").manual_seed(5))

    def f(x):
        return 3 * KLRef(s.double() + x * e, t.double(), None, 1.5).loss.item()
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    tol = 3 * (KLRef(s, t, None, 1.5).d_tol * e.abs()).sum().item() + 1e-6
    assert abs((d.double() * e).sum().item() - slope) <= tol


def test_same_bits_every_time_and_captured():
    x, y = logits(5, 40000, seed=1), logits(5, 40000, seed=2)
    ids = torch.arange(5, device="cuda")

    def once():
        r = token_logprobs(x, ids, 20)
        loss, a, b = logits_kl_forward(x, y)
        return [*r, loss, logits_kl_backward(x, y, a, b)]
    first = once()
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        held = once()
    x.copy_(logits(5, 40000, seed=3))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, once()))


def test_long_offsets():
    """A row that starts past 2^31 elements."""
    V, T = 65536, 33000
    x = torch.zeros(1, T, V, device="cuda", dtype=torch.bfloat16)
    x[0, -2:] = logits(2, V)
    ids = torch.full((1, T), 5, device="cuda")
    r = token_logprobs(x, ids, 3)
    ref = TokenRef(x[:, -2:], ids[:, -2:], 3)
    assert_within(r.logprob[:, -2:], ref.logprob, ref.logprob_tol, "logprob")
    assert torch.equal(r.top_indices[:, -2:], ref.top_indices)
    assert torch.equal(r.top_indices[0, 0], torch.arange(3, device="cuda"))
    leaf = x.requires_grad_(True)
    (d,) = torch.autograd.grad(token_logprobs(leaf, ids).logprob.sum(), leaf)
    want = TokenRef(x[:, -2:], ids[:, -2:], g=torch.ones(1, 2, device="cuda"))
    assert_within(d[:, -2:], want.d, want.d_tol, "d_logits")


def test_nothing_to_do():
    x = torch.empty(2, 0, 100, device="cuda", requires_grad=True)
    r = token_logprobs(x, torch.empty(2, 0, dtype=torch.int64, device="cuda"), 3)
    assert r.logprob.shape == (2, 0) and r.top_indices.shape == (2, 0, 3)
    loss = logits_kl_align(x, x.detach())
    assert loss.item() == 0
    loss.backward()
    assert x.grad.shape == x.shape


def test_no_second_derivative():
    x, y = logits(3, 50, dtype="fp32").requires_grad_(True), logits(3, 50, dtype="fp32", seed=1)
    for f in (lambda: token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda")).logprob.sum(),
              lambda: logits_kl_align(x, y)):
        (d,) = torch.autograd.grad(f(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum(), x)


def test_refusals():
    x = logits(2, 5, 100)
    ids = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    for a, b, kw in ((x.double(), ids, {}), (x, ids.int(), {}), (x, ids[:, :4], {}), (x, ids.cpu(), {}),
                     (x.transpose(1, 2), ids, {}), (x[None], ids[None], {}), (x, ids, dict(top_k=33)),
                     (x, ids, dict(top_k=-1)), (x[..., :3], ids, dict(top_k=4)),
                     (x, ids, dict(top_k=1.5)), (x, ids, dict(ignore_index=None))):
        with pytest.raises(AssertionError):
            token_logprobs(a, b, **kw)
    m = torch.ones(2, 5, device="cuda", dtype=torch.bool)
    for a, b, kw in ((x, x.float(), {}), (x, x[:, :4], {}), (x, x.cpu(), {}),
                     (x, x, dict(temperature=0.0)), (x, x, dict(temperature=float("nan"))),
                     (x, x, dict(temperature="1")), (x, x, dict(attn_mask=m[:, :4])),
                     (x, x, dict(attn_mask=m.float())), (x.transpose(1, 2), x.transpose(1, 2), {})):
        with pytest.raises(AssertionError):
            logits_kl_align(a, b, **kw)


def test_gradients_of_what_is_seen_twice():
    """The same row for the whole batch, and one tensor as student and teacher."""
    row = logits(1, 4, 300, dtype="fp32").requires_grad_(True)
    ids = torch.arange(8, device="cuda").view(2, 4)
    (d,) = torch.autograd.grad(token_logprobs(row.expand(2, -1, -1), ids).logprob.sum(), row)
    many = row.detach().expand(2, -1, -1).contiguous()
    ref = TokenRef(many, ids, g=torch.ones(2, 4, device="cuda"))
    assert_within(d, ref.d.sum(0, keepdim=True), ref.d_tol.sum(0, keepdim=True), "d_row")
    (d,) = torch.autograd.grad(logits_kl_align(row, row), row)
    assert (d == 0).all()
