"""End-to-end self-distillation step with the KL operator dropped in.

This is the training step of LinearARD's ``train.py:165-465`` for the
end-to-end benchmark configuration: a random-init LLaMA2-7B architecture
(32 layers, hidden 4096, 32 heads, d = 128, vocab 32000), uniform random
token ids, seq 16384, batch 1 per GPU; a frozen teacher with native RoPE and
a student with linear-scaled RoPE (factor 8) and LoRA r = 16 on q/k/v; the
loss is the Q/Q, K/K and V/V relation KL of every layer, normalised as
``train.py:380-410`` does; DDP over NCCL all-reduces the LoRA gradients.

What differs from the reference driver, in mechanism only:

* q/k/v are captured by an attention function registered with transformers
  (as ``record_qkv_attention``, ``train.py:109-145``) but kept as the views
  the attention layer produced: no ``.contiguous()`` copies
  (``attn_kl_align_grouped`` reads strided inputs in place);
* the 3·L relation losses are one grouped call instead of 3·L calls;
* LoRA is a small module written here (peft is not in this image): base
  weight frozen, ``A`` Kaiming-uniform, ``B`` zero, scale ``alpha / r``,
  no dropout (peft's defaults for these fields, ``train.py:271-273``);
* the model is ``LlamaModel`` without the LM head: the logits-KL term is off
  by default in the reference (``lam_l = 0``), so logits are not computed.
  ``--lam-l`` > 0 adds it (``train.py:413-423``): a frozen head that both
  models share, and ``lam_l`` times the mean KL of the tokens' distributions
  (``logits_kl_align``).  ``--token-metrics`` reports the student's next-token
  loss, entropy and accuracy on the sequence (``token_logprobs``);
* ``--attention own`` runs the models' attention on ``linearard_b200.attention``
  (forward and recomputing backward) instead of SDPA.

    python -m linearard_b200.distill [--layers 32] [--seq 16384] [--steps 3]
    torchrun --nproc-per-node 8 --master-addr 127.0.0.1 -m linearard_b200.distill

Prints one JSON line on rank 0 (tokens/s over all ranks, ms per step).
"""
from __future__ import annotations

import argparse
import json
import math
import os

import torch
import torch.distributed as dist
import torch.nn as nn

from .attention import attn
from .attention_KL import attn_kl_align_grouped
from .logits import logits_kl_align, token_logprobs

_ACTIVE = None   # the Capture the registered attention function records into


class Capture:
    """Per-layer q, k, v of one forward pass ([B, H, T, D] views)."""

    def __init__(self):
        self.q, self.k, self.v = {}, {}, {}

    def __enter__(self):
        global _ACTIVE
        _ACTIVE = self
        return self

    def __exit__(self, *exc):
        global _ACTIVE
        _ACTIVE = None

    def record(self, layer, q, k, v):
        self.q[layer], self.k[layer], self.v[layer] = q, k, v


# Options of transformers' attention interface that change its result and that `attn`
# does not have
_NOT_COMPUTED = ("softcap", "s_aux", "head_mask", "position_bias", "cu_seq_lens_q",
                 "cu_seq_lens_k")


def _check_mask_function(f, batch, q_length, kv_length, device):
    """Refuses a transformers mask function that removes more than the future (a window
    narrower than the sequence, packed sequences).  One that is neither of the plain two
    is evaluated, 1024 rows at a time."""
    from transformers.masking_utils import bidirectional_mask_function, causal_mask_function
    if f in (None, causal_mask_function, bidirectional_mask_function):
        return
    b, h, q, k = (torch.arange(n, device=device).view([-1 if i == d else 1 for i in range(4)])
                  for d, n in enumerate((batch, 1, q_length, kv_length)))
    causal = full = torch.ones((), dtype=torch.bool, device=device)
    for rows in q.split(1024, dim=2):
        keep = f(b, h, rows, k)
        causal = causal & (keep == (k <= rows)).all()
        full = full & keep.all()
    assert bool(causal | full), \
        "the attention takes causal or full masks, no windows or packed sequences"


def register_capture_attention(name=None, attention="sdpa"):
    """Register an attention implementation that records q, k, v (after
    RoPE, as the reference hook sees them) and then runs SDPA, or this package's
    attention (``attention="own"``: fp16 or bf16 on CUDA; a [B, T] padding mask
    removes tokens as queries and as keys; a sliding window narrower than the
    sequence, packed sequences, soft caps and sinks are refused)."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    assert attention in ("sdpa", "own"), "attention must be sdpa or own"
    name = name or ("lkl_capture" if attention == "sdpa" else "lkl_capture_own")

    def capture_attention(module, query, key, value, attention_mask, **kwargs):
        if _ACTIVE is not None:
            _ACTIVE.record(module.layer_idx, query, key, value)
        if attention == "sdpa":
            return sdpa_attention_forward(module, query, key, value, attention_mask, **kwargs)
        assert not kwargs.get("dropout"), "the attention has no dropout"
        window = kwargs.get("sliding_window")
        assert window is None or window >= key.shape[2], "the attention has no sliding window"
        for option in _NOT_COMPUTED:
            assert kwargs.get(option) is None, f"the attention has no {option}"
        assert attention_mask is None or attention_mask.ndim == 2, \
            "the attention takes [B, T] padding masks"
        causal = kwargs.get("is_causal")
        causal = getattr(module, "is_causal", True) if causal is None else causal
        if attention_mask is not None:
            attention_mask = attention_mask.contiguous()
        out = attn(query, key, value, attention_mask, causal, kwargs.get("scaling"))
        return out.transpose(1, 2), None

    def padding_mask(*args, attention_mask=None, mask_function=None, batch_size=None,
                     q_length=None, kv_length=None, device=None, **kwargs):
        assert not args, "the arguments of a mask function go by name"
        _check_mask_function(mask_function, batch_size, q_length, kv_length, device)
        return attention_mask            # [B, T]: the operator takes it as it is

    ALL_ATTENTION_FUNCTIONS.register(name, capture_attention)
    if attention == "own":
        ALL_MASK_ATTENTION_FUNCTIONS.register(name, padding_mask)
    return name


class LoRALinear(nn.Module):
    """y = base(x) + (x A^T B^T) * alpha / r, base frozen."""

    def __init__(self, base: nn.Linear, r: int, alpha: float):
        super().__init__()
        self.base = base
        for p in self.base.parameters():
            p.requires_grad_(False)
        dev, dt = base.weight.device, base.weight.dtype
        self.lora_A = nn.Parameter(torch.empty(r, base.in_features, device=dev, dtype=dt))
        self.lora_B = nn.Parameter(torch.zeros(base.out_features, r, device=dev, dtype=dt))
        nn.init.kaiming_uniform_(self.lora_A, a=math.sqrt(5))
        self.scale = alpha / r

    def forward(self, x):
        return self.base(x) + (x @ self.lora_A.t() @ self.lora_B.t()) * self.scale


def add_qkv_lora(model, r: int, alpha: float):
    for p in model.parameters():
        p.requires_grad_(False)
    for layer in model.layers:
        att = layer.self_attn
        att.q_proj = LoRALinear(att.q_proj, r, alpha)
        att.k_proj = LoRALinear(att.k_proj, r, alpha)
        att.v_proj = LoRALinear(att.v_proj, r, alpha)
    return [p for p in model.parameters() if p.requires_grad]


def llama_config(layers, hidden, heads, intermediate, vocab, seq, rope, attn):
    from transformers import LlamaConfig
    cfg = LlamaConfig(vocab_size=vocab, hidden_size=hidden, intermediate_size=intermediate,
                      num_hidden_layers=layers, num_attention_heads=heads,
                      num_key_value_heads=heads, max_position_embeddings=max(seq, 4096),
                      rope_parameters=rope)
    cfg._attn_implementation = attn
    cfg.use_cache = False
    return cfg


def build_models(args, device, seed=0):
    """Teacher (native RoPE, frozen) and student (same weights, linear RoPE x
    factor, LoRA on q/k/v), random init in bf16 on `device`."""
    from transformers import LlamaModel
    impl = register_capture_attention(attention=getattr(args, "attention", "sdpa"))
    base_rope = {"rope_type": "default", "rope_theta": args.rope_theta}
    student_rope = {"rope_type": "linear", "factor": args.rope_factor,
                    "rope_theta": args.rope_theta}
    torch.manual_seed(seed)
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(device):
            teacher = LlamaModel(llama_config(args.layers, args.hidden, args.heads,
                                              args.intermediate, args.vocab, args.seq,
                                              base_rope, impl))
            student = LlamaModel(llama_config(args.layers, args.hidden, args.heads,
                                              args.intermediate, args.vocab, args.seq,
                                              student_rope, impl))
    finally:
        torch.set_default_dtype(old)
    student.load_state_dict(teacher.state_dict())
    teacher.eval()
    for p in teacher.parameters():
        p.requires_grad_(False)
    lora = add_qkv_lora(student, args.lora_r, args.lora_alpha)
    student.train()
    return teacher, student, lora


def relation_loss(cap_s: Capture, cap_t: Capture, layers, attn_mask=None, sm_scale=None):
    """train.py:380-410: per layer KL_Q/denom + KL_K/denom + KL_V/denom, mean
    over layers, denom = valid tokens x Hq.  One grouped call for all of them."""
    items = []
    for l in layers:
        for s, t in ((cap_s.q[l], cap_t.q[l]), (cap_s.k[l], cap_t.k[l]),
                     (cap_s.v[l], cap_t.v[l])):
            items.append((s, s, t, t))
    kl = attn_kl_align_grouped(items, attn_mask=attn_mask, causal=True, sm_scale_s=sm_scale,
                               sm_scale_t=sm_scale)
    qs = cap_s.q[layers[0]]
    if attn_mask is None:
        denom = qs.shape[0] * qs.shape[1] * qs.shape[2]
    else:
        denom = attn_mask.sum().clamp_min(1) * qs.shape[1]
    return kl.sum() / denom / max(1, len(layers))


def build_head(args, device, seed=0):
    """The frozen LM head that both models share, random init in bf16."""
    g = torch.Generator(device=device).manual_seed(seed)
    head = nn.Linear(args.hidden, args.vocab, bias=False, device=device, dtype=torch.bfloat16)
    head.weight.data.normal_(0.0, 0.02, generator=g)
    return head.requires_grad_(False)


def logits_loss(logits_s, logits_t, attn_mask=None, temperature=1.0):
    """Mean over the valid tokens of KL(teacher || student) of their next-token
    distributions (the term that ``lam_l`` weighs, train.py:413-423)."""
    kl = logits_kl_align(logits_s, logits_t, attn_mask=attn_mask, temperature=temperature)
    if attn_mask is None:
        return kl / max(1, logits_s.shape[:-1].numel())
    return kl / attn_mask.sum().clamp_min(1)


def token_metrics(logits, input_ids, attn_mask=None):
    """The student's next-token loss, entropy and accuracy: position t answers
    token t + 1; positions whose next token is padding do not count."""
    targets = input_ids[:, 1:]
    if attn_mask is not None:
        targets = targets.masked_fill(attn_mask[:, 1:] == 0, -100)
    with torch.no_grad():
        r = token_logprobs(logits[:, :-1], targets, top_k=1)
        on = targets != -100
        n = on.sum().clamp_min(1)
        return {"nll": -r.logprob.sum() / n,
                "entropy": r.entropy.masked_fill(~on, 0.0).sum() / n,
                "accuracy": ((r.top_indices[..., 0] == targets) & on).sum() / n}


def parse(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=32)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--intermediate", type=int, default=11008)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--seq", type=int, default=16384)
    ap.add_argument("--rope-theta", type=float, default=10000.0)
    ap.add_argument("--rope-factor", type=float, default=8.0)
    ap.add_argument("--lora-r", type=int, default=16)
    ap.add_argument("--lora-alpha", type=float, default=32.0)
    ap.add_argument("--lr", type=float, default=1e-4)
    ap.add_argument("--attention", choices=("sdpa", "own"), default="sdpa")
    ap.add_argument("--lam-l", type=float, default=0.0)
    ap.add_argument("--temperature", type=float, default=1.0)
    ap.add_argument("--token-metrics", action="store_true")
    ap.add_argument("--steps", type=int, default=3)
    ap.add_argument("--warmup", type=int, default=1)
    return ap.parse_args(argv)


def main(argv=None):
    from torch.nn.parallel import DistributedDataParallel as DDP
    args = parse(argv)
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if world > 1:
        dist.init_process_group("nccl", device_id=dev)
    teacher, student, lora = build_models(args, dev, seed=0)
    model = DDP(student, device_ids=[local]) if world > 1 else student
    opt = torch.optim.AdamW(lora, lr=args.lr)
    layers = list(range(args.layers))
    g = torch.Generator(device=dev).manual_seed(1000 + rank)
    with_logits = args.lam_l > 0 or args.token_metrics
    head = build_head(args, dev) if with_logits else None
    tokens = {}

    def step(marks=None):
        def mark():
            if marks is not None:
                marks.append(torch.cuda.Event(enable_timing=True))
                marks[-1].record()
        ids = torch.randint(0, args.vocab, (1, args.seq), device=dev, generator=g)
        mark()
        with torch.no_grad(), Capture() as cap_t:
            out_t = teacher(input_ids=ids, use_cache=False)
        mark()
        with Capture() as cap_s:
            out_s = model(input_ids=ids, use_cache=False)
        mark()
        loss = relation_loss(cap_s, cap_t, layers)
        if with_logits:
            logits_s = head(out_s.last_hidden_state)
            if args.lam_l > 0:
                with torch.no_grad():
                    logits_t = head(out_t.last_hidden_state)
                loss = loss + args.lam_l * logits_loss(logits_s, logits_t,
                                                       temperature=args.temperature)
            if args.token_metrics:
                tokens.update(token_metrics(logits_s.detach(), ids))
        mark()
        loss.backward()                      # DDP all-reduces the LoRA gradients
        mark()
        opt.step()
        opt.zero_grad(set_to_none=True)
        mark()
        out = loss.detach()
        if world > 1:
            dist.all_reduce(out)
            out /= world
        return out

    for _ in range(args.warmup):
        step()
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(args.steps):
        loss = step()
    e1.record()
    torch.cuda.synchronize()
    ms = torch.tensor([e0.elapsed_time(e1) / args.steps], device=dev)
    # one more step with events between its phases (reported, not in the timing)
    marks = []
    step(marks)
    torch.cuda.synchronize()
    names = ("teacher_forward", "student_forward", "kl_forward_grouped",
             "backward_kl_model_and_lora_allreduce", "optimizer")
    phases = {n: marks[i].elapsed_time(marks[i + 1]) for i, n in enumerate(names)}
    if world > 1:
        dist.all_reduce(ms, op=dist.ReduceOp.MAX)
    if rank == 0:
        ms_step = float(ms.item())
        print(json.dumps({
            "metric": "self-distillation step tokens/s (LLaMA2-7B arch, random init, LoRA r=%d "
                      "on q/k/v, Q/Q+K/K+V/V KL over all layers)" % args.lora_r,
            "value": args.seq * world / (ms_step / 1e3), "unit": "tokens/s", "n_gpus": world,
            "ms_per_step": ms_step, "steps": args.steps, "warmup": args.warmup,
            "config": {"layers": args.layers, "hidden": args.hidden, "heads": args.heads,
                       "seq_len": args.seq, "batch_per_gpu": 1, "rope_factor": args.rope_factor,
                       "lora_r": args.lora_r, "parallelism": f"ddp{world}",
                       "attention": args.attention, "lam_l": args.lam_l},
            "loss": float(loss.item()),
            **({"tokens_rank0": {k: float(v) for k, v in tokens.items()}} if tokens else {}),
            "phase_ms_rank0": phases,
            "peak_mem_gb": torch.cuda.max_memory_allocated(dev) / 2**30,
        }), flush=True)
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
