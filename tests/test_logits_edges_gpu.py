"""Logits operators at the edges of what their arguments allow: rows without a target,
common offsets, outputs changed in place."""
import pytest
import torch

from linearard_b200.logits import logits_kl_align, logits_kl_forward, token_logprobs
from operator_refs import KLRef, assert_within
from test_logits_gpu import logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [5, 1003, 50257])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("entropy", [False, True])
def test_rows_without_a_target_have_no_gradient_whatever_they_hold(dtype, V, poison, entropy):
    x = logits(3, 4, V, dtype=dtype)
    ids = torch.full((3, 4), 1, device="cuda")
    ids[0, 1] = ids[2, 3] = -100
    clean = x.clone()
    x[0, 1] = poison
    x[2, 3, V // 2:] = poison

    def grad(x):
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, ids)
        loss = -r.logprob.sum()
        if entropy:              # of the rows that have a target
            loss = loss + r.entropy.masked_fill(ids == -100, 0.0).sum()
        return torch.autograd.grad(loss, leaf)[0]
    got, want = grad(x), grad(clean)
    assert (got[ids == -100] == 0).all()
    assert torch.equal(got[ids != -100], want[ids != -100])


@pytest.mark.parametrize("rows,V", [(3, 7), (5, 1003), (2, 40000), (700, 9001), (2000, 32000)])
@pytest.mark.parametrize("tau", [1.0, 1.7])
@pytest.mark.parametrize("offsets", [(1024.0, 0.0), (-512.0, 1024.0), (100.0, 100.0)])
def test_kl_loss_does_not_see_a_rows_offset(rows, V, tau, offsets):
    """A constant added to a row changes no distribution.  The logits are multiples of 2^-9
    below 64, so that the sums are exact and so are all differences from a row's maximum:
    the loss keeps its bits."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    t = (torch.randn(rows, V, device="cuda", generator=g) * 2).mul(512).round().div(512)
    s = t + (torch.randn(rows, V, device="cuda", generator=g) * 0.1).mul(512).round().div(512)
    want = logits_kl_forward(s, t, temperature=tau)[0]
    got = logits_kl_forward(s + offsets[0], t + offsets[1], temperature=tau)[0]
    assert torch.equal((s + offsets[0]) - offsets[0], s) and torch.equal((t + offsets[1]) - offsets[1], t)
    assert torch.equal(got, want)
    ref = KLRef(s, t, None, tau)
    assert_within(got, ref.loss, ref.loss_tol, "loss")


def test_kl_masked_vocabulary():
    """Entries that both models exclude by the type's lowest number, or by -inf, add nothing,
    wherever they stand; neither does a run of them before the first real logit."""
    for low in (torch.finfo(torch.float32).min, -torch.inf):
        t, s = logits(4, 9000, dtype="fp32", seed=1), logits(4, 9000, dtype="fp32", seed=2)
        kept = KLRef(s[:, 6000:], t[:, 6000:])
        s[:, :6000] = t[:, :6000] = low
        leaf = s.clone().requires_grad_(True)
        loss = logits_kl_align(leaf, t)
        tol = KLRef(s, t).loss_tol
        assert_within(loss, kept.loss, tol, "loss")
        d = torch.autograd.grad(loss, leaf)[0]
        assert (d[:, :6000] == 0).all() and torch.isfinite(d).all()
        # the teacher alone excludes them
        s[:, :6000] = logits(4, 6000, dtype="fp32", seed=3)
        ref = KLRef(s, t)
        assert_within(logits_kl_forward(s, t)[0], ref.loss, ref.loss_tol, "loss")


def test_token_outputs_changed_in_place():
    x = logits(3, 4, 1003)
    ids = torch.arange(12, device="cuda").view(3, 4)
    keep = (ids % 3 != 0)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, ids)
    want = torch.autograd.grad((r.logprob * 2 * keep).sum() + r.entropy.sum(), leaf)[0]
    r = token_logprobs(leaf, ids)
    entropy = r.entropy.detach().clone()
    loss = r.logprob.mul_(2.0).masked_fill_(~keep, 0.0).sum() + r.entropy.sum()
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
    assert torch.equal(r.entropy.detach(), entropy)


def grid(*shape, seed=0, scale=2.0):
    """Multiples of 2^-9 below 64, so that adding 1024 is exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).mul(512).round().div(512)


def p_error(x):
    """How far p may be from itself under an exact offset: the log probability and its
    multiple by log2(e) are rounded (2^-24 of their size, both times), so is e^ (2^-22)."""
    lp = torch.log_softmax(x.double(), -1)
    return lp.exp() * (lp.abs() * 2.0 ** -22 + 2.0 ** -20)


@pytest.mark.parametrize("rows,V", [(3, 7), (5, 1003), (40, 40000)])
@pytest.mark.parametrize("tau", [1.0, 1.7])
@pytest.mark.parametrize("offset", [1024.0, -512.0])
def test_gradients_do_not_see_a_rows_offset(rows, V, tau, offset):
    t, s = grid(rows, V), grid(rows, V, seed=1)

    def kl(s, t):
        leaf = s.clone().requires_grad_(True)
        return torch.autograd.grad(logits_kl_align(leaf, t, temperature=tau), leaf)[0].double()
    want = kl(s, t)
    tol = (p_error(s / tau) + p_error(t / tau)) / tau + 2.0 ** -22 * want.abs() + 1e-38
    assert_within(kl(s + offset, t), want, tol, "student shifted")
    assert_within(kl(s, t + offset), want, tol, "teacher shifted")
    ids = torch.arange(rows, device="cuda")

    def token(x):
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, ids)
        return torch.autograd.grad(r.logprob.sum() + 0.5 * r.entropy.sum(), leaf)[0].double()
    want = token(s)
    lp = torch.log_softmax(s.double(), -1)
    size = 1.0 + 0.5 * (lp.abs() + 12.0)       # |g + h (log p + H)| with H below log V
    tol = p_error(s) * size + lp.exp() * 2.0 ** -20 * size + 2.0 ** -22 * want.abs() + 1e-38
    assert_within(token(s + offset), want, tol, "token logits shifted")


@pytest.mark.parametrize("V", [7, 1000, 9001])
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_fp32_kl_gradient_of_near_models(V, tau):
    """Where the models are near, each element's gradient is exact relative to its own size but
    for what the row's log-sum-exps carry: two sums of V fp32 terms, in practice 2^-22 of each
    (their worst case, V / 128 + 7 roundings of 2^-24 and exponentials of 2^-20, in full)."""
    t = grid(64, V, seed=5)
    step = 2.0 ** -9 * torch.randint(-8, 9, (64, V), device="cuda",
                                     generator=torch.Generator(device="cuda").manual_seed(6))
    s = (t + step).requires_grad_(True)
    got = torch.autograd.grad(logits_kl_align(s, t, temperature=tau), s)[0].double()
    ps, pt = (torch.softmax(x.detach().double() / tau, -1) for x in (s, t))
    want = (ps - pt) / tau
    # relative: the probability, e^x - 1 and the product; absolute: the row's two sums
    lp = torch.log_softmax(t.double() / tau, -1)
    rel = lp.abs() * 2.0 ** -22 + 2.0 ** -19
    rows = 2 * ((V / 128 + 7) * 2.0 ** -24 + 2.0 ** -20)
    assert_within(got, want, rel * want.abs() + rows * pt / tau + 1e-38, "ds")
    # what the row's sums carry is one factor for the row: without it the relative bound holds
    shift = ((got - want) / (pt / tau)).median(-1, keepdim=True).values
    assert_within(got - shift * pt / tau, want, rel * (want.abs() + 2.0 ** -8 * pt / tau) + 1e-38,
                  "ds beside the row's common part")
