"""The operators beside the relation loss, as cases to measure: the attention of
the distillation step (forward and recomputing backward), the log probabilities
of given tokens (with entropy and top alternatives) and the KL loss between a
teacher's and a student's logits.

``listed()`` gives the fixed cases, ``draw(rng)`` more of the same ranges,
``prepare`` a case's inputs, ``run`` one pass, ``work`` the bytes and operations
it cannot do without and ``exact`` its outputs in 64 bits.  With ``own`` false,
``run`` computes the operators in elementary torch operations; with ``own`` true
it calls ``linearard_b200``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100       # target of a position that has no token to score


# ------------------------------------------------------------------ cases
def listed():
    attn = dict(op="attn", causal=True, mask=False, backward=True, layout="bthd")
    tok = dict(op="token", dtype="bf16", backward=False, shifted=False)
    kl = dict(op="kl", dtype="bf16", mask=False, temperature=1.0)
    return [
        # a smoke-test sequence: two heads, a handful of padded tokens; the time is launches
        dict(attn, name="attn tiny padded fp16", B=1, Hq=2, Hkv=2, T=8, D=16, dtype="fp16",
             mask=True, layout="bhtd"),
        # a padded batch of short sequences, bidirectional
        dict(attn, name="attn padded batch d64", B=4, Hq=8, Hkv=8, T=1000, D=64, dtype="fp16",
             mask=True, causal=False),
        # one layer of the end-to-end distillation step at the training context of 4096
        dict(attn, name="attn 4k 32 heads", B=1, Hq=32, Hkv=32, T=4096, D=128, dtype="bf16"),
        # a long sequence with four query heads to a key head, odd length
        dict(attn, name="attn 15k grouped heads", B=1, Hq=8, Hkv=2, T=15001, D=128, dtype="bf16"),
        # the frozen teacher's layer: forward alone, 32 query heads on 8 key heads
        dict(attn, name="attn teacher 8k", B=1, Hq=32, Hkv=8, T=8192, D=128, dtype="bf16",
             backward=False),
        # scoring the one token that was just sampled
        dict(tok, name="token single row", B=1, T=1, V=32000, dtype="fp32", top_k=5),
        # scoring an evaluation text under a large vocabulary, with 20 alternatives to each token
        dict(tok, name="token 2k rows top 20", B=1, T=2048, V=128256, top_k=20),
        # next-token loss of a training batch: the logits of all but the last position
        dict(tok, name="token training batch", B=2, T=2049, V=32000, top_k=0, backward=True,
             shifted=True),
        # a vocabulary of odd size: no row but the first starts on 16 bytes
        dict(tok, name="token odd vocabulary", B=3, T=333, V=50257, dtype="fp16", top_k=1,
             backward=True),
        # a few positions of a small model
        dict(kl, name="kl small", B=2, T=9, V=1000, dtype="fp32", mask=True),
        # the distillation step's sequence of 16384 tokens
        dict(kl, name="kl 16k sequence", B=1, T=16384, V=32000),
        # padded batch, softened distributions, odd vocabulary
        dict(kl, name="kl padded odd vocabulary", B=4, T=501, V=50257, mask=True, temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("attn", "attn", "token", "kl"))
    if op == "attn":
        D = rng.choice((8, 16, 32, 64, 64, 128, 128, 128))
        Hkv = rng.choice((1, 2, 3, 4, 8))
        Hq = Hkv * rng.choice((1, 1, 2, 4))
        backward = rng.random() < 0.75
        # a single token has no gradient with respect to q and k
        T = _log_int(rng, 2 if backward else 1, 12000)
        # no more work than the largest listed case
        B = _log_int(rng, 1, max(1, min(8, int(8 * 15001 ** 2 / (Hq * T * T)))))
        while B * Hq * T * T > 8 * 15001 ** 2:
            T = T * 3 // 4
        return dict(op="attn", B=B, Hq=Hq, Hkv=Hkv, T=T, D=D, dtype=rng.choice(("bf16", "fp16")),
                    causal=rng.random() < 0.75, mask=rng.random() < 0.35,
                    backward=backward, layout=rng.choice(("bhtd", "bthd")))
    V = _log_int(rng, 500, 160000)
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    rows = _log_int(rng, 1, max(2, min(16000, int(2.6e8 / V))))
    B = rng.choice((1, 1, 2, 3))
    T = max(1, rows // B)
    if op == "token":
        return dict(op="token", B=B, T=T + 1, V=V, dtype=dtype, top_k=rng.choice((0, 1, 5, 20, 32)),
                    backward=rng.random() < 0.5, shifted=rng.random() < 0.5)
    return dict(op="kl", B=B, T=T, V=V, dtype=dtype, mask=rng.random() < 0.5,
                temperature=rng.choice((1.0, 1.0, 2.0, 0.7)))


# ------------------------------------------------------------------ inputs
def _padding(case, gen):
    """[B, T] int64, 1 = token: the rows are padded on the right up to a third."""
    B, T = case["B"], case["T"]
    short = torch.randint(0, T // 3 + 1, (B, 1), device="cuda", generator=gen)
    return (torch.arange(T, device="cuda")[None, :] < T - short).long()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, T = case["B"], case["T"]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).mul_(scale)

    state = dict(case)
    if case["op"] == "attn":
        def heads(n, scale):
            if case["layout"] == "bthd":   # a projection's output, seen as [B, H, T, D]
                x = randn(B, T, n, case["D"], scale=scale).to(dt).transpose(1, 2)
            else:
                x = randn(B, n, T, case["D"], scale=scale).to(dt)
            return x
        state["q"] = heads(case["Hq"], 1.3)
        state["k"] = heads(case["Hkv"], 1.3)
        state["v"] = heads(case["Hkv"], 1.0)
        state["attn_mask"] = _padding(case, gen) if case["mask"] else None
        if case["backward"]:
            state["dout"] = heads(case["Hq"], 1.0)
            for n in ("q", "k", "v"):
                state[n].requires_grad_(True)
        return state
    V = case["V"]
    x = randn(B, T, V, scale=2.0)
    if case["op"] == "token":
        ids = torch.randint(0, V, (B, T), device="cuda", generator=gen)
        x.scatter_add_(2, ids[..., None], randn(B, T, 1, scale=2.0) + 6.0)   # a model that knows
        state["logits"] = x.to(dt)
        if case["shifted"]:       # position t answers token t + 1
            state["logits"] = state["logits"][:, :-1]
            ids = ids[:, :-1]
        ids = ids.contiguous()
        ids.view(-1)[3::7] = IGNORE     # some positions have no target
        state["targets"] = ids
        if case["backward"]:
            state["logits"].requires_grad_(True)
            state["d_logprob"] = randn(*ids.shape)
            state["d_entropy"] = randn(*ids.shape, scale=0.1)
        return state
    state["teacher"] = x.to(dt)
    state["student"] = (x + randn(B, T, V, scale=0.5)).to(dt).requires_grad_(True)
    state["attn_mask"] = _padding(case, gen) if case["mask"] else None
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return {"attn": _attn, "token": _token, "kl": _kl}[state["op"]](state)


def _attn(s):
    if own:
        from linearard_b200.attention import attn, attn_forward
        args = dict(attn_mask=s["attn_mask"], causal=s["causal"])
        if not s["backward"]:
            out, lse = attn_forward(s["q"], s["k"], s["v"], **args)
            return {"out": out, "lse": lse}
        out = attn(s["q"], s["k"], s["v"], **args)
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        dt, B, T, D = s["q"].dtype, s["B"], s["T"], s["D"]
        Hq, Hkv = s["Hq"], s["Hkv"]
        G, sc = Hq // Hkv, D ** -0.5
        q = s["q"].float().reshape(B, Hkv, G * T, D)
        k, v = s["k"].float(), s["v"].float()
        x = (q @ k.transpose(-1, -2)).mul_(sc).view(B, Hkv, G, T, T)
        keep = torch.ones(1, 1, 1, T, T, dtype=torch.bool, device=q.device)
        if s["causal"]:
            keep = keep.tril()
        rows = None
        if s["attn_mask"] is not None:
            m = s["attn_mask"] != 0
            rows = m[:, None, None, :, None]
            keep = keep & m[:, None, None, None, :] & rows
        x.masked_fill_(~keep, float("-inf"))
        top = x.amax(-1, keepdim=True).clamp_min_(-1e30)
        p = x.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(total.clamp_min(1e-30))
        out = (p.view(B, Hkv, G * T, T) @ v).view(B, Hq, T, D)
        if not s["backward"]:
            lse = (top + total.log()).view(B, Hq, T)
            if rows is not None:
                lse = lse.masked_fill(~rows[:, :, 0, :, 0], 0.0)
            return {"out": out.to(dt), "lse": lse}
        do = s["dout"].float().reshape(B, Hkv, G * T, D)
        dv = p.view(B, Hkv, G * T, T).transpose(-1, -2) @ do
        dp = (do @ v.transpose(-1, -2)).view(B, Hkv, G, T, T)
        delta = (do.view(B, Hq, T, D) * out).sum(-1).view(B, Hkv, G, T, 1)
        ds = dp.sub_(delta).mul_(p).mul_(sc).view(B, Hkv, G * T, T)
        dq = (ds @ k).view(B, Hq, T, D)
        dk = ds.transpose(-1, -2) @ q
        return {"out": out.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


def _token(s):
    if own:
        from linearard_b200.logits import token_logprobs
        r = token_logprobs(s["logits"], s["targets"], top_k=s["top_k"], ignore_index=IGNORE)
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if s["top_k"]:
            out.update(top_logprobs=r.top_logprobs, top_indices=r.top_indices)
        if s["backward"]:
            out["d_logits"], = torch.autograd.grad((r.logprob, r.entropy), s["logits"],
                                                   (s["d_logprob"], s["d_entropy"]))
        return out
    with torch.no_grad():
        x = s["logits"].float()
        ids = s["targets"]
        some = ids != IGNORE
        at = torch.where(some, ids, 0)[..., None]
        logp = x - x.amax(-1, keepdim=True)
        logp -= logp.exp().sum(-1, keepdim=True).log()
        p = logp.exp()
        entropy = -(p * logp).sum(-1)
        chosen = torch.where(some, logp.gather(-1, at)[..., 0], 0.0)
        out = {"logprob": chosen, "entropy": entropy}
        if s["top_k"]:
            # by the logits as they are: equal ones keep their order
            order = s["logits"].sort(dim=-1, descending=True, stable=True).indices
            out["top_indices"] = order[..., :s["top_k"]].contiguous()
            out["top_logprobs"] = logp.gather(-1, out["top_indices"])
        if s["backward"]:
            g = torch.where(some, s["d_logprob"], 0.0)[..., None]
            h = s["d_entropy"][..., None]
            d = -p * (g + h * (logp + entropy[..., None]))
            d.scatter_add_(-1, at, g)
            out["d_logits"] = d.to(s["logits"].dtype)
        return out


def _kl(s):
    if own:
        from linearard_b200.logits import logits_kl_align
        loss = logits_kl_align(s["student"], s["teacher"], attn_mask=s["attn_mask"],
                               temperature=s["temperature"])
        grad, = torch.autograd.grad(loss, s["student"])
        return {"loss": loss, "d_student": grad}
    with torch.no_grad():
        # the loss is a small difference of long sums: 64 bits
        inv = 1.0 / s["temperature"]
        a, b = s["student"].double().mul_(inv), s["teacher"].double().mul_(inv)
        a -= a.amax(-1, keepdim=True)
        b -= b.amax(-1, keepdim=True)
        a -= a.exp().sum(-1, keepdim=True).log()
        b -= b.exp().sum(-1, keepdim=True).log()
        pt = b.exp()
        rows = (pt * b.sub_(a)).sum(-1)
        grad = a.exp_().sub_(pt).mul_(inv)
        if s["attn_mask"] is not None:
            keep = s["attn_mask"] != 0
            rows = rows * keep
            grad = grad * keep[..., None]
        return {"loss": rows.sum().float(), "d_student": grad.to(s["student"].dtype)}


# ------------------------------------------------------------------ least work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, T = case["B"], case["T"]
    if case["op"] == "attn":
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        pairs = B * Hq * (T * (T + 1) // 2 if case["causal"] else T * T)
        q, kv = B * Hq * T * D * size, B * Hkv * T * D * size
        nbytes = 2 * q + 2 * kv                         # q, k, v -> out
        flops = 4 * pairs * D
        if case["backward"]:
            nbytes += 4 * q + 4 * kv                    # q, k, v, dout again -> dq, dk, dv
            flops += 10 * pairs * D
        else:
            nbytes += B * Hq * T * 4
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "token":
        rows = B * (T - 1 if case["shifted"] else T)
        nbytes = rows * (case["V"] * size + 8 + 8 + 12 * case["top_k"])
        flops = 4 * rows * case["V"]
        if case["backward"]:
            nbytes += rows * (2 * case["V"] * size + 8)
            flops += 6 * rows * case["V"]
        return {"bytes": nbytes, "flops": flops}
    n = B * T * case["V"]
    # both logits for the loss; both again, and the gradient, afterwards
    return {"bytes": 5 * n * size, "flops": 16 * n}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "token": _exact_token, "kl": _exact_kl}[case["op"]](s)


def _exact_attn(s):
    B, T, G = s["B"], s["T"], s["Hq"] // s["Hkv"]
    scale = 1.0 / math.sqrt(s["D"])
    out = torch.zeros(B, s["Hq"], T, s["D"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, s["Hq"], T, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk = torch.zeros(B, s["Hkv"], T, s["D"], dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    for b in range(B):
        live = torch.arange(T, device="cuda")
        if s["attn_mask"] is not None:
            live = live[s["attn_mask"][b] != 0]
        for h in range(s["Hq"]):
            q, k, v = (s[n][b, i].double()[live] for n, i in (("q", h), ("k", h // G),
                                                             ("v", h // G)))
            w = torch.einsum("id,jd->ij", q, k) * scale
            if s["causal"]:
                w = w.masked_fill(live[None, :] > live[:, None], -math.inf)
            z = torch.logsumexp(w, 1)
            p = torch.exp(w - z[:, None])
            del w
            o = p @ v
            out[b, h, live], lse[b, h, live] = o, z
            if s["backward"]:
                g = s["dout"][b, h].double()[live]
                t = (g @ v.T - (g * o).sum(1, keepdim=True)) * p
                dq[b, h, live] = t @ k * scale
                dk[b, h // G, live] += t.T @ q * scale
                dv[b, h // G, live] += p.T @ g
    if not s["backward"]:
        return {"out": out, "lse": lse}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_token(s):
    outs = {}
    lp, en, grads, top = [], [], [], []
    for b in range(s["logits"].shape[0]):
        logp = torch.log_softmax(s["logits"][b].double(), dim=-1)
        p = torch.softmax(s["logits"][b].double(), dim=-1)
        ent = torch.special.entr(p).sum(-1)
        ids = s["targets"][b]
        rows = torch.nonzero(ids != IGNORE)[:, 0]
        picked = torch.zeros(len(ids), dtype=torch.float64, device="cuda")
        picked[rows] = logp[rows, ids[rows]]
        lp.append(picked)
        en.append(ent)
        if s["top_k"]:
            top.append(torch.topk(logp, s["top_k"], dim=-1).values)
        if s["backward"]:
            dl, de = s["d_logprob"][b].double(), s["d_entropy"][b].double()
            hot = torch.zeros_like(p)
            hot[rows, ids[rows]] = 1.0
            seen = torch.zeros_like(dl)
            seen[rows] = dl[rows]
            g = seen[:, None] * (hot - p)
            g -= de[:, None] * torch.where(p > 0, p * (logp + ent[:, None]), 0.0)
            grads.append(g)
    outs["logprob"], outs["entropy"] = torch.stack(lp), torch.stack(en)
    if s["top_k"]:
        outs["top_logprobs"], outs["top_indices"] = torch.stack(top), None
    if s["backward"]:
        outs["d_logits"] = torch.stack(grads)
    return outs


def _exact_kl(s):
    tau = s["temperature"]
    loss, grads = 0.0, []
    for b in range(s["B"]):
        ls = torch.log_softmax(s["student"][b].double() / tau, dim=-1)
        lt = torch.log_softmax(s["teacher"][b].double() / tau, dim=-1)
        row = torch.special.xlogy(lt.exp(), lt.exp()).sum(-1) - (lt.exp() * ls).sum(-1)
        g = (ls.exp() - lt.exp()) / tau
        if s["attn_mask"] is not None:
            off = s["attn_mask"][b] == 0
            row[off] = 0.0
            g[off] = 0.0
        loss = loss + row.sum()
        grads.append(g)
    return {"loss": loss, "d_student": torch.stack(grads)}
