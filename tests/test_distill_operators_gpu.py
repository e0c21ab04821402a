"""The distillation step with its own attention, the logits term and the token
metrics: a run of the operators together, against the step on SDPA and against
torch's log_softmax on the same logits."""
import contextlib
import io
import json

import pytest
import torch

from gpu_util import assert_grad_close, assert_loss_close, check_device_status
from linearard_b200 import distill

pytestmark = pytest.mark.gpu

SMALL = ["--layers", "2", "--hidden", "512", "--heads", "4", "--intermediate", "1024", "--vocab",
         "1003", "--seq", "520"]


def build(extra=(), seed=3):
    a = distill.parse(SMALL + list(extra))
    dev = torch.device("cuda", 0)
    teacher, student, lora = distill.build_models(a, dev, seed=seed)
    g = torch.Generator(device=dev).manual_seed(4)
    for m in student.modules():            # non-zero B so that every LoRA factor gets a gradient
        if isinstance(m, distill.LoRALinear):
            m.lora_B.data.normal_(0, 0.02, generator=g)
    ids = torch.randint(0, a.vocab, (2, a.seq), device=dev, generator=g)
    return a, teacher, student, lora, distill.build_head(a, dev), ids


def step(a, teacher, student, head, ids, mask=None):
    layers = list(range(a.layers))
    with torch.no_grad(), distill.Capture() as ct:
        ht = teacher(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
    with distill.Capture() as cs:
        hs = student(input_ids=ids, attention_mask=mask, use_cache=False).last_hidden_state
    ls, lt = head(hs), head(ht)
    loss = distill.relation_loss(cs, ct, layers, mask) + 0.5 * distill.logits_loss(ls, lt, mask, 1.5)
    return loss, ls, lt


def test_step_on_own_attention_matches_sdpa():
    """Both attentions round their probabilities to bf16, so the steps agree to the
    bar that the step's gradients are held to."""
    grads, losses = [], []
    for extra in ([], ["--attention", "own"]):
        a, teacher, student, lora, head, ids = build(extra)
        loss, _, _ = step(a, teacher, student, head, ids)
        loss.backward()
        losses.append(float(loss.detach()))
        grads.append([p.grad.float().cpu().numpy() for p in lora])
    check_device_status()
    assert_loss_close(losses[1], losses[0], rel=1e-2)
    for i, (x, y) in enumerate(zip(*grads)):
        assert_grad_close(y, x, f"lora[{i}]", rel_max=5e-2)


def test_padded_batch_ignores_padding():
    """What stands in the padding changes neither loss nor gradients."""
    a, teacher, student, lora, head, ids = build(["--attention", "own"])
    mask = torch.ones_like(ids)
    mask[1, 300:] = 0
    got = []
    for fill in (5, 900):
        x = ids.masked_fill(mask == 0, fill)
        for p in lora:
            p.grad = None
        loss, ls, _ = step(a, teacher, student, head, x, mask)
        loss.backward()
        got.append((loss.detach(), [p.grad.clone() for p in lora],
                    distill.token_metrics(ls.detach(), x, mask)))
    assert torch.equal(got[0][0], got[1][0])
    for x, y in zip(got[0][1], got[1][1]):
        assert torch.equal(x, y)
    for k in got[0][2]:
        assert torch.equal(got[0][2][k], got[1][2][k]), k
    check_device_status()


def test_logits_term_and_metrics_against_log_softmax():
    a, teacher, student, lora, head, ids = build(["--attention", "own"])
    _, ls, lt = step(a, teacher, student, head, ids)
    mask = torch.ones_like(ids)
    mask[0, 400:] = 0
    leaf = ls.detach().requires_grad_(True)
    loss = distill.logits_loss(leaf, lt, mask, 1.5)
    loss.backward()
    x = ls.detach().double().requires_grad_(True)
    p, q = torch.log_softmax(x / 1.5, -1), torch.log_softmax(lt.double() / 1.5, -1)
    ref = ((q.exp() * (q - p)).sum(-1) * mask).sum() / mask.sum()
    ref.backward()
    assert_loss_close(float(loss), float(ref), rel=1e-4, abs_=1e-7)
    # the gradient is rounded to bf16 (half a step: 2^-8), its probabilities are fp32
    assert ((leaf.grad.double() - x.grad).abs() <= 2.0 ** -8 * x.grad.abs() + 1e-9).all()
    m = distill.token_metrics(ls.detach(), ids, mask)
    lp = torch.log_softmax(ls.detach()[:, :-1].double(), -1)
    on = mask[:, 1:].bool()
    nll = -lp.gather(-1, ids[:, 1:, None])[..., 0][on].mean()
    ent = -(lp.exp() * lp).sum(-1)[on].mean()
    acc = (ls[:, :-1].float().argmax(-1) == ids[:, 1:])[on].double().mean()
    for k, v in (("nll", nll), ("entropy", ent), ("accuracy", acc)):
        assert_loss_close(float(m[k]), float(v), rel=1e-5, abs_=1e-6, name=k)


def test_command_reports_logits_loss_and_tokens():
    out = io.StringIO()
    with contextlib.redirect_stdout(out):
        distill.main(SMALL + ["--steps", "1", "--warmup", "1", "--attention", "own", "--lam-l", "0.5",
                              "--token-metrics"])
    line = json.loads(out.getvalue().strip().splitlines()[-1])
    assert line["config"]["attention"] == "own" and line["config"]["lam_l"] == 0.5
    assert line["loss"] > 0 and set(line["tokens_rank0"]) == {"nll", "entropy", "accuracy"}
    check_device_status()
