"""Gradients under saved-tensor hooks, which may give the saved tensors back in
another layout: the same bits as without hooks."""
import pytest
import torch

from gpu_util import check_device_status
from linearard_b200.attention import attn
from linearard_b200.logits import logits_kl_align, token_logprobs

pytestmark = pytest.mark.gpu


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def strange(t):
    """The same values with a last stride other than 1."""
    return torch.stack([t, t], -1)[..., 0] if t.ndim else t


def shifted(t):
    """The same values and strides, one element off a 16-byte boundary."""
    if not t.is_floating_point() or not t.is_contiguous():
        return t
    return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)


HOOKS = {
    "cpu": lambda: torch.autograd.graph.save_on_cpu(pin_memory=False),
    "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    **{f.__name__: (lambda f=f: torch.autograd.graph.saved_tensors_hooks(lambda t: t, f))
       for f in (dense, strange, shifted)},
}


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("layout", ["bthd", "fused", "bhtd"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention(hook, layout, D):
    B, Hq, Hkv, T = 2, 4, 2, 200
    g = torch.Generator(device="cuda").manual_seed(D)

    def heads(H):
        if layout == "bhtd":
            return torch.randn(B, H, T, D, device="cuda", generator=g).bfloat16()
        n = 2 * D if layout == "fused" else D
        x = torch.randn(B, T, H, n, device="cuda", generator=g).bfloat16()
        return x[..., -D:].transpose(1, 2)
    q, k, v = (heads(H).requires_grad_(True) for H in (Hq, Hkv, Hkv))
    dout = heads(Hq)
    mask = torch.ones(B, T, device="cuda", dtype=torch.int64)
    mask[1, 150:] = 0
    want = torch.autograd.grad(attn(q, k, v, mask), (q, k, v), dout)
    with HOOKS[hook]():
        out = attn(q, k, v, mask)
    got = torch.autograd.grad(out, (q, k, v), dout)
    torch.cuda.synchronize()
    check_device_status()
    for name, a, b in zip("qkv", got, want):
        assert torch.equal(a, b), name


CUTS = {"shift": lambda x: x[:, :-1], "vocab": lambda x: x[..., 3:998], "rows": lambda x: x[1],
        "whole": lambda x: x}


def logits(cut, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(3, 9, 1003, device="cuda", generator=g).to(dtype)
    return CUTS[cut](x)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs(hook, cut, dtype):
    x = logits(cut, dtype, 1).requires_grad_(True)
    ids = torch.arange(x.shape[:-1].numel(), device="cuda").view(x.shape[:-1]) * 7 % x.shape[-1]

    def grads(context):
        with context():
            r = token_logprobs(x, ids)
        return torch.autograd.grad(r.logprob.sum() + 0.3 * r.entropy.sum(), x)[0]
    want = grads(lambda: torch.enable_grad())
    assert torch.equal(grads(HOOKS[hook]), want)


@pytest.mark.parametrize("hook", HOOKS)
@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [False, True])
def test_logits_kl(hook, cut, dtype, mask):
    s, t = logits(cut, dtype, 1).requires_grad_(True), logits(cut, dtype, 2)
    m = torch.ones(s.shape[:-1], device="cuda", dtype=torch.int64) if mask else None
    if mask:
        m[..., 5:] = 0

    def grads(context):
        with context():
            loss = logits_kl_align(s, t, m, 1.5)
        return torch.autograd.grad(loss, s)[0]
    want = grads(lambda: torch.enable_grad())
    assert torch.equal(grads(HOOKS[hook]), want)
