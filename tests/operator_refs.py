"""Plain float64 formulations of the attention and logits operators, and how far
a kernel may be from them.

The bounds follow from the arithmetic, not from runs.  u = eps / 2 of the
tensors' 16-bit type is the largest relative error of one rounding.  A score is
an fp32 sum of D products: off by at most D 2^-24 sum |q||k| sc; its exponent
is rounded once more (2^-23 of its size) and an fp32 exponential or logarithm
is off by less than 2^-20.  P and dS may be rounded to 16 bits before their
products, whose fp32 sums are off by n 2^-24 of the sum of magnitudes.
"""
import torch


class AttnRef:
    """Attention and its gradients in float64, with elementwise bounds."""

    def __init__(self, q, k, v, mask=None, causal=True, sc=None, dout=None):
        u, q16 = torch.finfo(q.dtype).eps / 2, q.dtype
        B, Hq, T, D = q.shape
        G = Hq // k.shape[1]
        sc = D ** -0.5 if sc is None else sc
        keep = torch.ones(B, 1, T, T, dtype=torch.bool, device=q.device)
        if causal:
            keep = keep.tril()
        live = torch.ones(B, T, dtype=torch.bool, device=q.device)
        if mask is not None:
            live = mask.to(q.device) != 0
        keep = keep & live[:, None, None, :] & live[:, None, :, None]
        rows = live[:, None, :, None]

        def clean(x, rep=1):      # what a removed token holds takes no part
            x = torch.where(rows, x.detach().double(), 0.0)
            return x.repeat_interleave(rep, 1)

        q, k, v = clean(q), clean(k, G), clean(v, G)
        S = (q @ k.transpose(-1, -2)) * sc
        mag = (q.abs() @ k.abs().transpose(-1, -2)) * sc
        S = torch.where(keep, S, -torch.inf)
        self.lse = torch.where(rows[..., 0], torch.logsumexp(S, -1), 0.0)
        P = torch.where(keep, torch.exp(S - self.lse[..., None]), 0.0)
        acc = (T + 32) * 2.0 ** -24
        # relative error of a probability: its score, and the row's log-sum-exp
        top = torch.where(keep, mag, 0.0).amax(-1, keepdim=True)
        c = 2 * (D * 2.0 ** -24 + 2.0 ** -22) * top + 2.0 ** -19 + acc
        self.lse_tol = (c[..., 0] + 2.0 ** -22 * self.lse.abs())
        self.out = P @ v
        self.out_tol = u * self.out.abs() + (1 + u) * (u + c + acc) * (P @ v.abs()) + 1e-30
        if dout is None:
            return
        g = clean(dout)
        dP = g @ v.transpose(-1, -2)
        delta = (g * self.out).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        # delta is taken with the rounded output
        d_delta = (g.abs() * (self.out_tol + D * 2.0 ** -24 * self.out.abs())).sum(-1, keepdim=True)
        d_dp = D * 2.0 ** -24 * (g.abs() @ v.abs().transpose(-1, -2))
        dS_tol = (u + c) * dS.abs() + (1 + u) * P * (d_delta + d_dp + 2.0 ** -22 *
                                                     (dP.abs() + delta.abs()))
        # below the normal numbers a rounding is off by half of the smallest step: 2^-25
        # in fp16.  bf16 has the exponents of fp32, whose kernels may flush what is
        # below 2^-126 to zero
        tiny = 2.0 ** -25 if q16 == torch.float16 else 2.0 ** -126
        dS_tol = dS_tol + torch.where(keep, tiny, 0.0)
        P_tol = (u + c + acc) * P + torch.where(keep, tiny, 0.0)
        self.out_tol = self.out_tol + tiny * v.abs().sum(-2, keepdim=True) + tiny

        def heads(x):             # sums over the query heads of a kv head
            return x.view(B, Hq // G, G, T, D).sum(2)

        self.dq = sc * dS @ k
        self.dq_tol = sc * (dS_tol + acc * dS.abs()) @ k.abs() * (1 + u) + u * self.dq.abs() + tiny
        acc_g = (G * T + 32) * 2.0 ** -24
        self.dk = heads(sc * dS.transpose(-1, -2) @ q)
        self.dk_tol = (heads(sc * (dS_tol + acc_g * dS.abs()).transpose(-1, -2) @ q.abs()) * (1 + u)
                       + u * self.dk.abs() + tiny)
        self.dv = heads(P.transpose(-1, -2) @ g)
        self.dv_tol = (heads((P_tol + acc_g * P).transpose(-1, -2) @ g.abs()) * (1 + u)
                       + u * self.dv.abs() + tiny)


def assert_within(got, ref, tol, name):
    got = got.detach().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name} is not finite"
    over = (got - ref).abs() - tol
    worst = over.max().item() if over.numel() else 0.0
    at = over.argmax().item() if over.numel() else 0
    assert worst <= 0, (f"{name}: off by {(got - ref).abs().flatten()[at]:.3e} at {at}, allowed "
                        f"{tol.flatten()[at]:.3e} (value {ref.flatten()[at]:.3e})")


def row_tol(x, V):
    """Absolute error that fp32 statistics of a row of V logits may carry into
    its log-sum-exp: the sum of V exponentials (each off by 2^-20, its exponent
    rounded by 2^-23 of its size), accumulated by some hundred threads, and the
    roundings of the result."""
    spread = (x.amax(-1) - x.clamp_min(-1e4).amin(-1)).clamp_max(100.0)
    size = x.amax(-1).abs() + torch.logsumexp(x, -1).abs()
    return (V / 64 + 64) * 2.0 ** -24 + 2.0 ** -20 + spread * 2.0 ** -23 + size * 2.0 ** -22


class TokenRef:
    def __init__(self, logits, targets, top_k=0, ignore=-100, g=None, h=None):
        x = logits.detach().double()
        V = x.shape[-1]
        lse = torch.logsumexp(x, -1)
        tol = row_tol(x, V)
        lp = x - lse[..., None]
        p = lp.exp()
        plp = torch.where(p > 0, p * lp, 0.0)
        hit = targets != ignore
        at = torch.where(hit, targets, 0)[..., None]
        self.logprob = torch.where(hit, lp.gather(-1, at)[..., 0], 0.0)
        self.logprob_tol = tol
        self.entropy = -plp.sum(-1)
        # sum e (x - m): the relative errors above on terms of size |x - m|
        self.entropy_tol = tol * (2 + (p * (x - x.amax(-1, keepdim=True)).abs().nan_to_num(0.0, posinf=0.0)).sum(-1))
        order = logits.detach().sort(dim=-1, descending=True, stable=True).indices[..., :top_k]
        self.top_indices, self.top_logprobs = order, lp.gather(-1, order)
        if g is not None or h is not None:
            u = 0.0 if logits.dtype == torch.float32 else torch.finfo(logits.dtype).eps / 2
            u = max(u, 2.0 ** -23)
            g = torch.zeros_like(lse) if g is None else torch.where(hit, g.double(), 0.0)
            h = torch.zeros_like(lse) if h is None else h.double()
            hot = torch.zeros_like(p).scatter_(-1, at, hit[..., None].double())
            self.d = g[..., None] * (hot - p) - h[..., None] * (plp + p * self.entropy[..., None])
            mag = g.abs()[..., None] * (hot + p) + h.abs()[..., None] * (plp.abs() + p * self.entropy[..., None])
            rel = 2 * tol[..., None] + 2.0 ** -19
            self.d_tol = (u * self.d.abs() + rel * mag
                          + h.abs()[..., None] * p * (tol + self.entropy_tol)[..., None]
                          + (2.0 ** -25 if logits.dtype == torch.float16 else 1e-38))


class KLRef:
    def __init__(self, s, t, mask=None, tau=1.0):
        a, b = s.detach().double() / tau, t.detach().double() / tau
        V = a.shape[-1]
        on = torch.ones(a.shape[:-1], dtype=torch.bool, device=a.device)
        if mask is not None:
            on = mask.to(a.device) != 0
        ls, lt = torch.log_softmax(a, -1), torch.log_softmax(b, -1)
        pt, ps = lt.exp(), ls.exp()
        rows = torch.where(pt > 0, pt * (lt - ls), 0.0).sum(-1)
        diff = (pt * torch.where(pt > 0, b - a, 0.0).abs()).sum(-1)
        # the weighted sum and the two log-sum-exps carry relative errors; the
        # maxima and their difference are exact in 64 bits
        rel = (V / 64 + 64) * 2.0 ** -24 + 2.0 ** -20 + 100 * 2.0 ** -23
        row_err = rel * (2 + diff) + rows.abs() * 2.0 ** -23
        self.loss = torch.where(on, rows, 0.0).sum()
        self.loss_tol = torch.where(on, row_err, 0.0).sum() + self.loss.abs() * 2.0 ** -23
        self.lse_s = torch.where(on, torch.logsumexp(a, -1), 0.0)
        self.lse_t = torch.where(on, torch.logsumexp(b, -1), 0.0)
        u = 2.0 ** -23 if s.dtype == torch.float32 else torch.finfo(s.dtype).eps / 2
        self.d = torch.where(on[..., None], (ps - pt) / tau, 0.0)
        err = (2 * torch.maximum(row_tol(a, V), row_tol(b, V))[..., None] + 2.0 ** -19) * (ps + pt)
        self.d_tol = u * self.d.abs() + torch.where(on[..., None], err / tau, 0.0) + (
            2.0 ** -25 if s.dtype == torch.float16 else 1e-38)
