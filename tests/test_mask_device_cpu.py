"""A padding mask on another GPU than the tensors is refused before its address goes to
a kernel: fake CUDA tensors, no GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from linearard_b200.attention import attn, attn_backward, attn_forward
from linearard_b200.attention_KL import attn_kl_align, attn_kl_align_grouped, attn_kl_align_strided
from linearard_b200.attention_KL._common import prepare_mask
from linearard_b200.logits import logits_kl_align, logits_kl_backward, logits_kl_forward


def test_mask_on_another_gpu():
    with FakeTensorMode():
        q = torch.empty(2, 4, 64, 64, device="cuda:0", dtype=torch.bfloat16)
        lse = torch.empty(2, 4, 64, device="cuda:0")
        x, rows = torch.empty(2, 64, 100, device="cuda:0"), torch.empty(2, 64, device="cuda:0")
        mask = torch.ones(2, 64, device="cuda:1", dtype=torch.int64)
        for call in (lambda: attn(q, q, q, mask), lambda: attn_forward(q, q, q, mask),
                     lambda: attn_backward(q, q, q, q, q, lse, mask),
                     lambda: logits_kl_align(x, x, mask), lambda: logits_kl_forward(x, x, mask),
                     lambda: logits_kl_backward(x, x, rows, rows, mask),
                     lambda: attn_kl_align(q, q, q, q, mask),
                     lambda: attn_kl_align_strided(q, q, q, q, mask),
                     lambda: attn_kl_align_grouped([(q, q, q, q)], mask)):
            with pytest.raises(AssertionError, match="attn_mask must be on the device"):
                call()
        assert prepare_mask(mask.to("cuda:0"), 2, 64, q.device)[0].device == q.device
