"""Logits operators at the edges of what their arguments allow: rows without a target,
common offsets, outputs changed in place."""
import pytest
import torch

from linearard_b200.logits import logits_kl_align, logits_kl_forward, token_logprobs
from operator_refs import TokenRef, assert_within
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
