"""float64 attention over contexts with the bounds that the tests hold the kernels to (helpers of tests/test_gpu_context_attention*.py).

Tolerance of an output o = sum p v / sum p whose probabilities p are rounded once to the storage type (u = finfo.eps / 2):
    u |o|                              the result's own rounding
    u sum p |v| / sum p                every p off by u relative (the sum itself is kept in fp32)
    2^-25 sum |v| / sum p              fp16 only: a p below 2^-14 is a subnormal, off by half of 2^-24 (the largest p of a part is 1)
    2 e sum p |v| / sum p              e: relative error of p from the fp32 scores, 2^-24 (d + 32) scale max sum |q k| + 2^-21 (exp2 and rescaling)

Tolerance of the gradients, with ds = p (dp - D), dp = do v^T, D = sum do o:
    dv: u |dv| + (u + 4 e) p^T |do|                                 p rounded once; its error now includes the saved log-sum-exp's
    ds: (u + 4 e) |ds| + p (sum |do| tol(o)) + 2^-24 (d + 8) p (|do| |v|^T + sum |do o|)        rounded once; D is taken from the rounded o
        + 2^-37 (max|dp| + max|D|) in fp16                          (p is carried as 2^12 p, dp - D with a power of two of at least 1 / its maximum: off by half a subnormal step)
    dq: u |dq| + scale tol(ds) |k|,   dk: u |dk| + scale tol(ds)^T |q|,   each plus half a subnormal step of fp16
"""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def split(t, heads):
    return t.detach().double().cpu().reshape(t.shape[0], t.shape[1], heads, t.shape[2] // heads).transpose(1, 2)      # [B, heads, N, d]


def live_keys(B, Nq, Np, Nk, lens, mask, causal):
    """[B, Nq, Np + Nk] truth values."""
    n = torch.full((B,), Nk) if lens is None else lens.cpu().long().clamp(0, Nk)
    at = torch.arange(Nk)
    own = (at < n.view(B, 1, 1)).expand(B, Nq, Nk)
    if causal:
        own = own & (at <= (n.view(B, 1, 1) - Nq + torch.arange(Nq).view(1, Nq, 1)))
    if mask is not None:
        own = own & mask.cpu().view(-1, 1, Nk)
    return torch.cat([torch.ones(B, Nq, Np, dtype=torch.bool), own], 2)


class Reference:
    """o, lse and the tolerance of o for q [B, Nq, H d], k / v [B or 1, Nk, Hk d], prefix [Np, Hk d]; dead keys are taken as zeros."""

    def __init__(self, q, k, v, heads, kv_heads=None, lens=None, mask=None, scale=None, k_prefix=None, v_prefix=None, causal=False):
        kv_heads = kv_heads or heads
        B, Nq = q.shape[:2]
        self.dtype, self.heads, self.kv_heads, self.d = q.dtype, heads, kv_heads, q.shape[2] // heads
        self.scale = self.d ** -0.5 if scale is None else scale
        Np = 0 if k_prefix is None else k_prefix.shape[0]
        rep = heads // kv_heads
        self.q = split(q, heads)
        ks, vs = (split(t, kv_heads).expand(B, -1, -1, -1) for t in (k, v))
        if Np:
            ks, vs = (torch.cat([split(p[None], kv_heads).expand(B, -1, -1, -1), t], 2) for p, t in ((k_prefix, ks), (v_prefix, vs)))
        self.live = live_keys(B, Nq, Np, k.shape[1], lens, mask, causal).unsqueeze(1)
        dead = ~self.live.any(2).squeeze(1).view(B, 1, -1, 1)
        self.k, self.v = (t.masked_fill(dead, 0.0).repeat_interleave(rep, 1) for t in (ks, vs))
        s = (self.q @ self.k.transpose(2, 3) * self.scale).masked_fill(~self.live, -math.inf)
        m = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:3], 1), -math.inf, dtype=s.dtype)
        e = torch.exp(s - m.clamp_min(-1e300)).masked_fill(~self.live, 0.0)
        total = e.sum(-1, keepdim=True)
        self.p = e / total.clamp_min(1e-300)
        self.o = self.p @ self.v
        self.lse = (m + torch.log(total)).squeeze(-1)
        u = U[self.dtype]
        self.e = 2.0 ** -24 * (self.d + 32) * self.scale * float((self.q.abs() @ self.k.abs().transpose(2, 3)).max() if s.numel() else 0) + 2.0 ** -21
        av = self.p @ self.v.abs()
        self.tol = u * self.o.abs() + (u + 2 * self.e) * av + 1e-30
        if self.dtype == torch.float16:
            self.tol = self.tol + 2.0 ** -25 * (self.live.double() @ self.v.abs()) / total.clamp_min(1.0) * (total > 0) + 2.0 ** -25

    def check(self, out, lse=None, what=""):
        got = split(out, self.heads)
        bad = ~((got - self.o).abs() <= self.tol)
        assert not bad.any(), f"{what} out: {int(bad.sum())} of {bad.numel()} outside, worst {((got - self.o).abs() / self.tol).max():.3g} of the tolerance"
        if lse is not None:
            g = lse.double().cpu()
            none = torch.isinf(self.lse)
            assert torch.equal(none, torch.isinf(g)) and (g[none] < 0).all()
            err = (g - self.lse).abs()[~none]
            assert (err <= 2 * self.e + 2.0 ** -22 * (1 + self.lse[~none].abs())).all(), f"{what} lse: worst {err.max():.3g}"

    def check_gradients(self, dout, dq, dk, dv, shared, what=""):
        B, H, Nq, Nk = self.p.shape
        go = split(dout, self.heads)
        u = U[self.dtype]
        sub = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        dp = go @ self.v.transpose(2, 3)
        D = (go * self.o).sum(-1, keepdim=True)
        ds = self.p * (dp - D)
        r_dv, t_dv = self.p.transpose(2, 3) @ go, (u + 4 * self.e) * (self.p.transpose(2, 3) @ go.abs())
        t_ds = (u + 4 * self.e) * ds.abs() + self.p * (go.abs() * self.tol).sum(-1, keepdim=True) + \
            2.0 ** -24 * (self.d + 8) * self.p * (go.abs() @ self.v.abs().transpose(2, 3) + (go * self.o).abs().sum(-1, keepdim=True))
        t_ds = (t_ds + 2.0 ** -12 * sub * float(dp.abs().max() + D.abs().max())) * self.live
        r_dq, t_dq = self.scale * (ds @ self.k), self.scale * (t_ds @ self.k.abs())
        r_dk, t_dk = self.scale * (ds.transpose(2, 3) @ self.q), self.scale * (t_ds.transpose(2, 3) @ self.q.abs())

        def fold(t):                                                               # heads of a group, and the batch where one context serves it
            t = t.view(B, self.kv_heads, H // self.kv_heads, Nk, self.d).sum(2)
            return t.sum(0, keepdim=True) if shared else t
        for n, got, r, t, heads in (("dq", dq, r_dq, t_dq, H), ("dk", dk, fold(r_dk), fold(t_dk), self.kv_heads), ("dv", dv, fold(r_dv), fold(t_dv), self.kv_heads)):
            if got is None:
                continue
            g = split(got, heads)
            tol = t + u * r.abs() + sub + 1e-30
            bad = ~((g - r).abs() <= tol)
            assert not bad.any(), f"{what} {n}: {int(bad.sum())} of {bad.numel()} outside, worst {((g - r).abs() / tol).max():.3g} of the tolerance"
            if n != "dq":
                dead = ~self.live.any(2)[:, 0]                                     # [B, Nk]
                dead = dead.all(0, keepdim=True) if shared else dead
                assert not got[dead.to(got.device)].any(), f"{what} {n}: a key that does not exist has a gradient"


def randn(shape, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)
