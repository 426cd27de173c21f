"""Measured cases of the operators around the UNet's contexts: GroupNorm with an activation on channels-last maps, cross attention to
an encoder's states of another length, and attention of a batch that shares one long prefix of keys.

`own` false: `run` computes the operators from elementary torch operations in fp32 (rounded once at the end); `own` true: it makes the
calls of `vidseg_diffusion_amd.ops`.  Both take what `prepare` returns.  Keys:

    op         "norm" | "cross" | "prefix"
    dir        "infer": the forward pass; "train": the forward pass and the gradients of every differentiable input
    dtype      storage type of maps, queries, keys and values (norm parameters are fp32, lengths int32)
    batch      samples; queries / keys: tokens per sample; prefix: keys that all samples share
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # the deepest map of the SD 2.1 UNet for one CFG pair, fp32 as the exact mode keeps it: a call that latency decides
        dict(name="norm_train_f32_8x8", op="norm", dir="train", dtype="float32", batch=2, height=8, width=8, channels=1280, groups=32, silu=True),
        # first level of the SD 2.1 UNet at 512 x 512, 14 frames with both CFG halves: the largest map of a ResBlock
        dict(name="norm_infer_f16_64x64", op="norm", dir="infer", dtype="float16", batch=28, height=64, width=64, channels=320, groups=32, silu=True),
        # the decoder's concatenated map (1280 + 640 channels) at 32 x 32 while the network is tuned on 14 frames
        dict(name="norm_train_bf16_32x32", op="norm", dir="train", dtype="bfloat16", batch=14, height=32, width=32, channels=1920, groups=32, silu=True),
        # a transformer's entrance norm (no activation) on the 56 x 104 latent of a wide clip
        dict(name="norm_train_f16_56x104", op="norm", dir="train", dtype="float16", batch=14, height=56, width=104, channels=320, groups=32, silu=False),
        # one pooled query per image over the ViT-H tower's 257 tokens, heads of 80
        dict(name="cross_infer_bf16_pool", op="cross", dir="infer", dtype="bfloat16", batch=8, queries=1, keys=257, heads=16, kv_heads=16, head_dim=80, shared=False),
        # text cross attention of the first UNet level: 4096 tokens against prompts of up to 77 tokens, padded to different lengths
        dict(name="cross_infer_f16_text", op="cross", dir="infer", dtype="float16", batch=28, queries=4096, keys=77, heads=5, kv_heads=5, head_dim=64, shared=False),
        # the same layer one level deeper while prompt embeddings and projections are tuned; one prompt for all frames
        dict(name="cross_train_bf16_text", op="cross", dir="train", dtype="bfloat16", batch=14, queries=1024, keys=77, heads=10, kv_heads=10, head_dim=64, shared=True),
        # tuning against a long encoder sequence (image tokens of another resolution), odd lengths
        dict(name="cross_train_f16_long", op="cross", dir="train", dtype="float16", batch=4, queries=1456, keys=2311, heads=10, kv_heads=10, head_dim=64, shared=False),
        # grouped heads of 128 over several thousand encoder states
        dict(name="cross_train_bf16_grouped", op="cross", dir="train", dtype="bfloat16", batch=2, queries=4096, keys=4096, heads=16, kv_heads=4, head_dim=128, shared=False),
        # one new token for each of four captions behind a prompt of 77 tokens
        dict(name="prefix_token_f16_small", op="prefix", dir="infer", dtype="float16", batch=4, queries=1, prefix=77, keys=33, heads=16, kv_heads=16, head_dim=64, causal=True),
        # one new token for each of 64 sequences that share a prompt of 16 K tokens, grouped heads
        dict(name="prefix_token_bf16", op="prefix", dir="infer", dtype="bfloat16", batch=64, queries=1, prefix=16384, keys=512, heads=32, kv_heads=8, head_dim=128, causal=True),
        # the tokens of 14 frames over an anchor frame's keys and their own
        dict(name="prefix_frames_f16", op="prefix", dir="infer", dtype="float16", batch=14, queries=4096, prefix=4096, keys=4096, heads=5, kv_heads=5, head_dim=64, causal=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "cross", "prefix"])
    if op == "norm":
        while True:
            groups = rng.choice([8, 16, 32])
            c = dict(op="norm", dir=rng.choice(["infer", "train"]), dtype=rng.choice(["float16", "bfloat16", "float32"]), batch=_log(rng, 1, 28),
                     height=_log(rng, 4, 104), width=_log(rng, 4, 104), channels=groups * _log(rng, 4, 60), groups=groups,
                     silu=rng.random() < 0.6)
            if c["batch"] * c["height"] * c["width"] * c["channels"] <= 28 * 64 * 64 * 320:
                return c
    kv = rng.choice([1, 2, 4, 5, 8, 10])
    group = rng.choice([1, 1, 1, 2, 4])
    base = dict(dtype=rng.choice(["float16", "bfloat16"]), heads=kv * group, kv_heads=kv)
    if op == "cross":
        while True:
            c = dict(op="cross", dir=rng.choice(["infer", "train"]), batch=_log(rng, 1, 28), queries=_log(rng, 1, 4096), keys=_log(rng, 1, 4096),
                     head_dim=rng.choice([40, 64, 80, 128]), shared=rng.random() < 0.25, **base)
            if c["batch"] * c["heads"] * c["queries"] * c["keys"] * c["head_dim"] <= 2 * 16 * 4096 * 4096 * 128:
                return c
    while True:
        few = rng.random() < 0.6
        c = dict(op="prefix", dir="infer", batch=_log(rng, 1, 64), queries=rng.choice([1, 1, 1, 2, 5]) if few else _log(rng, 16, 4096),
                 prefix=_log(rng, 16, 16384), keys=_log(rng, 8, 4096), head_dim=rng.choice([64, 80, 128]), causal=few, **base)
        c["keys"] = max(c["keys"], c["queries"]) if few else c["keys"]
        if c["batch"] * c["heads"] * c["queries"] * (c["prefix"] + c["keys"]) * c["head_dim"] <= 14 * 5 * 4096 * 8192 * 64 \
                and c["batch"] * c["keys"] * c["kv_heads"] * c["head_dim"] <= 64 * 4096 * 4 * 128:
            return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * scale + shift).to(dtype)

    s = dict(case=case)
    train = case["dir"] == "train"
    B = case["batch"]
    if case["op"] == "norm":
        C = case["channels"]
        # maps of a trained network: channel means apart from zero, some channels much louder than others
        loud = torch.exp(0.5 * torch.randn(C, generator=g, device=dev))
        mean = torch.randn(C, generator=g, device=dev)
        x = torch.randn(B, case["height"], case["width"], C, generator=g, device=dev)
        s["x"] = (x * loud + mean).to(dt)
        s["gamma"] = normal(C, scale=0.3, shift=1.0, dtype=torch.float32)
        s["beta"] = normal(C, scale=0.3, dtype=torch.float32)
        leaves = ("x", "gamma", "beta")
        s["dout"] = normal(*s["x"].shape, scale=0.1) if train else None
    else:
        H, Hk, d, Nq, Nk = case["heads"], case["kv_heads"], case["head_dim"], case["queries"], case["keys"]
        s["q"] = normal(B, Nq, H * d, scale=1.5)
        Bk = 1 if case.get("shared") else B
        s["k"] = normal(Bk, Nk, Hk * d)
        s["v"] = normal(Bk, Nk, Hk * d)
        low = max(min(Nk, Nq) if case.get("causal") else 1, Nk // 2)                       # sequences of different lengths, padded to the longest
        lens = torch.randint(low, Nk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        lens[0] = Nk
        s["lens"] = lens
        if case["op"] == "prefix":
            s["k_prefix"] = normal(case["prefix"], Hk * d)
            s["v_prefix"] = normal(case["prefix"], Hk * d)
        leaves = ("q", "k", "v")
        s["dout"] = normal(B, Nq, H * d, scale=0.1) if train else None
    if train:
        for n in leaves:
            s[n].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------- plain forms: elementary operations in fp32
def _plain_norm(s):
    c = s["case"]
    B, C, G = c["batch"], c["channels"], c["groups"]
    dt = s["x"].dtype
    x = s["x"].detach().float().view(B, -1, G, C // G)
    gamma, beta = s["gamma"].detach().view(G, C // G), s["beta"].detach().view(G, C // G)
    n = x.shape[1] * (C // G)
    mean = x.sum((1, 3), keepdim=True) / n
    xc = x - mean
    rstd = 1 / ((xc * xc).sum((1, 3), keepdim=True) / n + EPS).sqrt()
    xh = xc * rstd
    z = xh * gamma + beta
    sig = 1 / (1 + (-z).exp())
    out = z * sig if c["silu"] else z
    out = out.to(dt).view_as(s["x"])
    if c["dir"] == "infer":
        return out
    dz = s["dout"].float().view(x.shape)
    if c["silu"]:
        dz = dz * (sig * (1 + z * (1 - sig)))
    dbeta = dz.sum((0, 1)).view(C)
    dgamma = (dz * xh).sum((0, 1)).view(C)
    dxh = dz * gamma
    dx = rstd * (dxh - (dxh.sum((1, 3), keepdim=True) + xh * (dxh * xh).sum((1, 3), keepdim=True)) / n)
    return out, dx.to(dt).view_as(s["x"]), dgamma, dbeta


def _rows(x, B, N, Hk, G, d):
    """[B, N, Hk * G * d] -> fp32 [B, Hk, N * G, d]: the queries that read one key head, as the rows of one product."""
    return x.detach().float().view(B, N, Hk, G, d).permute(0, 2, 1, 3, 4).reshape(B, Hk, N * G, d)


def _back(x, B, N, Hk, G, d):
    return x.view(B, Hk, N, G, d).permute(0, 2, 1, 3, 4).reshape(B, N, Hk * G * d)


def _heads(x, Hk, d):
    """[B, N, Hk * d] -> fp32 [B, Hk, N, d]."""
    return x.detach().float().view(x.shape[0], x.shape[1], Hk, d).transpose(1, 2).contiguous()


def _softmax(sc):
    m = sc.amax(-1, keepdim=True)
    e = (sc - m.clamp_min(-1e30)).exp()
    total = e.sum(-1, keepdim=True)
    return e / total.clamp_min(1e-30)


def _plain_cross(s):
    c = s["case"]
    B, Nq, Nk, H, Hk, d = c["batch"], c["queries"], c["keys"], c["heads"], c["kv_heads"], c["head_dim"]
    G, scale, dt = H // Hk, d ** -0.5, s["q"].dtype
    q = _rows(s["q"], B, Nq, Hk, G, d)
    k, v = (_heads(s[n], Hk, d).expand(B, Hk, Nk, d) for n in ("k", "v"))
    live = torch.arange(Nk, device=q.device) < s["lens"].view(B, 1, 1, 1)
    p = _softmax((q @ k.transpose(2, 3) * scale).masked_fill(~live, -math.inf))
    out = _back(p @ v, B, Nq, Hk, G, d).to(dt)
    if c["dir"] == "infer":
        return out
    do = _rows(s["dout"], B, Nq, Hk, G, d)
    dv = p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = _back(ds @ k, B, Nq, Hk, G, d).to(dt)
    dk = ds.transpose(2, 3) @ q
    if c["shared"]:
        dk, dv = dk.sum(0, keepdim=True), dv.sum(0, keepdim=True)
    dk, dv = (t.transpose(1, 2).reshape(t.shape[0], Nk, Hk * d).to(dt) for t in (dk, dv))
    return out, dq, dk, dv


def _plain_prefix(s):
    c = s["case"]
    B, Nq, Np, Nk, H, Hk, d = c["batch"], c["queries"], c["prefix"], c["keys"], c["heads"], c["kv_heads"], c["head_dim"]
    G, scale = H // Hk, d ** -0.5
    q = _rows(s["q"], B, Nq, Hk, G, d) * scale
    k, v = _heads(s["k"], Hk, d), _heads(s["v"], Hk, d)
    kp, vp = _heads(s["k_prefix"][None], Hk, d)[0], _heads(s["v_prefix"][None], Hk, d)[0]
    last = s["lens"].view(B, 1, 1).expand(B, Nq, 1)                                            # keys that a query may see: those before it
    if c["causal"]:
        last = last - (Nq - 1 - torch.arange(Nq, device=q.device)).view(1, Nq, 1)
    live = (torch.arange(Nk, device=q.device) < last).repeat_interleave(G, 1).unsqueeze(1)     # [B, 1, Nq * G, Nk]
    qp = q.transpose(0, 1).reshape(Hk, B * Nq * G, d)                                          # the prefix is read once for the whole batch
    sp = (qp @ kp.transpose(1, 2)).view(Hk, B, Nq * G, Np)
    so = (q @ k.transpose(2, 3)).masked_fill(~live, -math.inf).transpose(0, 1)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = (sp - m).exp(), (so - m).exp()
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    o = (ep.view(Hk, B * Nq * G, Np) @ vp).view(Hk, B, Nq * G, d) + eo @ v.transpose(0, 1)
    return _back((o / total).transpose(0, 1).contiguous(), B, Nq, Hk, G, d).to(s["q"].dtype)


def _own(s):
    from vidseg_diffusion_amd import ops
    c = s["case"]
    if c["op"] == "norm":
        out = ops.groupnorm_act(s["x"], s["gamma"], s["beta"], groups=c["groups"], eps=EPS, act=ops.ACT_SILU if c["silu"] else ops.ACT_NONE)
        wrt = ("x", "gamma", "beta")
    elif c["op"] == "cross":
        out = ops.cross_attention(s["q"], s["k"], s["v"], c["heads"], kv_heads=c["kv_heads"], k_lens=s["lens"])
        wrt = ("q", "k", "v")
    else:
        return ops.prefix_attention(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], c["heads"], kv_heads=c["kv_heads"],
                                    k_lens=s["lens"], causal=c["causal"])
    if c["dir"] == "infer":
        return out
    return (out.detach(), *torch.autograd.grad(out, [s[n] for n in wrt], s["dout"]))


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "cross": _plain_cross, "prefix": _plain_prefix}[state["case"]["op"]](state)


def work(case):
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    train = c["dir"] == "train"
    B = c["batch"]
    if c["op"] == "norm":
        n = B * c["height"] * c["width"] * c["channels"]
        return {"bytes": n * size * (4 if train else 2), "flops": n * (30 if train else 12)}
    H, Hk, d, Nq = c["heads"], c["kv_heads"], c["head_dim"], c["queries"]
    keys = 0.75 * c["keys"]                                                                    # lengths spread over [keys / 2, keys]
    rows = B * Nq * H * d * size
    kv = 2 * (1 if c.get("shared") else B) * keys * Hk * d * size
    if c["op"] == "cross":
        return {"bytes": rows * (4 if train else 2) + kv * (2 if train else 1), "flops": B * H * Nq * keys * d * (14 if train else 4)}
    return {"bytes": 2 * rows + kv + 2 * c["prefix"] * Hk * d * size, "flops": 4 * B * H * Nq * (keys + c["prefix"]) * d}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    train = c["dir"] == "train"
    f64 = lambda t: t.detach().double().requires_grad_(train)                                  # noqa: E731
    if c["op"] == "norm":
        outs, dxs = [], []
        gamma, beta = f64(s["gamma"]), f64(s["beta"])
        dgamma, dbeta = torch.zeros_like(gamma), torch.zeros_like(beta)
        for b in range(c["batch"]):
            x = f64(s["x"][b])
            t = x.reshape(-1, c["groups"], c["channels"] // c["groups"])
            var, mean = torch.var_mean(t, dim=(0, 2), unbiased=False, keepdim=True)
            z = ((t - mean) / torch.sqrt(var + EPS)).reshape(x.shape) * gamma + beta
            y = z * torch.sigmoid(z) if c["silu"] else z
            outs.append(y.detach())
            if train:
                gx, gg, gb = torch.autograd.grad(y, (x, gamma, beta), s["dout"][b].double())
                dxs.append(gx)
                dgamma, dbeta = dgamma + gg, dbeta + gb
        return (torch.stack(outs), torch.stack(dxs), dgamma, dbeta) if train else torch.stack(outs)
    B, Nq, H, Hk, d = c["batch"], c["queries"], c["heads"], c["kv_heads"], c["head_dim"]
    if train and 14 * B * H * Nq * c["keys"] * d > 4e12 or 4 * B * H * Nq * (c["keys"] + c.get("prefix", 0)) * d > 4e12:
        return None
    out = torch.empty(B, Nq, H, d, dtype=torch.float64, device=s["q"].device)
    dq = torch.empty_like(out) if train else None
    dk = torch.zeros(s["k"].shape[0], c["keys"], Hk, d, dtype=torch.float64, device=out.device) if train else None
    dv = torch.zeros_like(dk) if train else None
    lens = s["lens"].tolist()
    for b in range(B):
        bk = 0 if c.get("shared") else b
        n = lens[b]
        for h in range(H):
            hk = h // (H // Hk)
            q = f64(s["q"][b, :, h * d:(h + 1) * d])
            k, v = (f64(s[t][bk, :n, hk * d:(hk + 1) * d]) for t in ("k", "v"))
            ka, va = k, v
            if c["op"] == "prefix":
                ka, va = (torch.cat([s[t + "_prefix"][:, hk * d:(hk + 1) * d].double(), own_t]) for t, own_t in (("k", k), ("v", v)))
            sc = q @ ka.T / math.sqrt(d)
            if c.get("causal"):
                seen = c["prefix"] + n - Nq + torch.arange(Nq, device=out.device)
                sc = sc.masked_fill(torch.arange(sc.shape[1], device=out.device)[None] > seen[:, None], -math.inf)
            o = torch.softmax(sc, -1) @ va
            out[b, :, h] = o.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["dout"][b, :, h * d:(h + 1) * d].double())
                dq[b, :, h] = gq
                dk[bk, :n, hk] += gk
                dv[bk, :n, hk] += gv
    if not train:
        return out.reshape(B, Nq, H * d)
    return out.reshape(B, Nq, H * d), dq.reshape(B, Nq, H * d), dk.reshape(dk.shape[0], -1, Hk * d), dv.reshape(dv.shape[0], -1, Hk * d)
