"""Gradients of ops.cross_attention against float64 (bounds: tests/tools_context_attention.py) and against differences."""
import os
import sys

import pytest
import torch

from vidseg_diffusion_amd import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from tools_context_attention import Reference, randn  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def step(q, k, v, heads, dout, **how):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, heads, **how)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


CASES = [  # B, Nq, Nk, H, Hk, d, dtype, lens, shared
    (2, 64, 77, 5, 5, 64, F16, None, False),                    # one pass for all three gradients (up to 128 keys)
    (3, 130, 77, 2, 2, 64, BF16, (77, 1, 0), False),
    (1, 1, 1, 1, 1, 8, F16, None, False),
    (4, 100, 77, 3, 3, 64, BF16, (77, 30, 1, 0), True),         # one context, lengths by sample, gradients summed over the batch
    (3, 65, 128, 4, 2, 128, F16, (128, 127, 0), True),
    (2, 90, 96, 2, 2, 80, BF16, (96, 33), False),
    (2, 31, 65, 4, 1, 40, F16, (64, 65), False),                # a group of 4 heads
    (2, 33, 129, 3, 3, 96, F16, (129, 128), False),             # more than 128 keys: two passes
    (1, 257, 300, 6, 2, 104, BF16, (300,), False),
    (2, 257, 200, 4, 2, 128, F16, (128, 0), True),
    (1, 700, 1031, 1, 1, 24, F16, None, False),
    (2, 1, 400, 8, 2, 128, BF16, (400, 77), False),
    (1, 2000, 50, 1, 1, 64, BF16, None, False),                 # rows in several chunks, partial sums joined
    (2, 40, 0, 2, 2, 64, F16, None, False),
    (1, 128, 128, 2, 2, 64, BF16, None, False),
]


@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,dtype,lens,shared", CASES)
def test_gradients(B, Nq, Nk, H, Hk, d, dtype, lens, shared):
    dev = torch.device("cuda:0")
    q, dout = randn((B, Nq, H * d), 1, dtype, 1.5).to(dev), randn((B, Nq, H * d), 6, dtype, 0.1).to(dev)
    k, v = (randn((1 if shared else B, Nk, Hk * d), s, dtype).to(dev) for s in (2, 3))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out, dq, dk, dv = step(q, k, v, H, dout, kv_heads=Hk, k_lens=n)
    with torch.no_grad():
        assert torch.equal(out, ops.cross_attention(q, k, v, H, kv_heads=Hk, k_lens=n))
    ref = Reference(q, k, v, H, Hk, n)
    ref.check(out)
    if Nk:
        ref.check_gradients(dout, dq, dk, dv, shared and B > 1)
    else:
        assert not dq.any() and dk.shape == k.shape
    again = step(q, k, v, H, dout, kv_heads=Hk, k_lens=n)
    assert all(torch.equal(a, b) for a, b in zip((out, dq, dk, dv), again))


@pytest.mark.parametrize("Nk,shared", [(100, False), (100, True), (330, False), (330, True)])
def test_mask_and_poison(Nk, shared):
    """Keys that do not exist: no gradient, and NaN or infinities there change no bit of any gradient."""
    dev = torch.device("cuda:0")
    B, Nq, H, d = 3, 70, 2, 64
    for dtype in (F16, BF16):
        q, dout = randn((B, Nq, H * d), 1, dtype).to(dev), randn((B, Nq, H * d), 6, dtype, 0.1).to(dev)
        k, v = (randn((1 if shared else B, Nk, H * d), s, dtype).to(dev) for s in (2, 3))
        g = torch.Generator().manual_seed(4)
        mask = torch.rand((B, Nk), generator=g) < 0.5
        mask[1] = False
        mask[:, 10:20] = False
        mask = mask.to(dev)
        lens = torch.tensor([Nk, Nk, Nk - 31], dtype=torch.int32, device=dev)
        got = step(q, k, v, H, dout, k_lens=lens, key_mask=mask)
        Reference(q, k, v, H, None, lens, mask).check_gradients(dout, *got[1:], shared)
        assert not got[1][1].any()                                                # the sample without a key
        exists = mask & (torch.arange(Nk, device=dev) < lens.view(B, 1))
        dead = ~(exists.any(0, keepdim=True) if shared else exists)
        for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
            k2, v2 = (t.masked_fill(dead.unsqueeze(-1), bad) for t in (k, v))
            assert all(torch.equal(a, b) for a, b in zip(got, step(q, k2, v2, H, dout, k_lens=lens, key_mask=mask)))


@pytest.mark.parametrize("Nk", [77, 200])
def test_gradient_scales(Nk):
    """fp16 output gradients from 2^-14 to 2^10, and rows of very different size: the intermediate gradient stays in range."""
    dev = torch.device("cuda:0")
    q, k, v = (randn((2, n, 128), s, F16).to(dev) for n, s in ((100, 1), (Nk, 2), (Nk, 3)))
    for power in (-14, 0, 10):
        dout = (randn((2, 100, 128), 6, torch.float32, 0.5) * 2.0 ** power).to(F16).to(dev)
        got = step(q, k, v, 2, dout)
        Reference(q, k, v, 2).check_gradients(dout, *got[1:], False, f"2^{power}")
    dout = (randn((2, 100, 128), 6, torch.float32) * torch.logspace(-4, 2, 100).view(1, 100, 1)).to(F16).to(dev)
    got = step(q, k, v, 2, dout)
    Reference(q, k, v, 2).check_gradients(dout, *got[1:], False, "rows")
    zero = step(q, k, v, 2, torch.zeros_like(dout))
    assert not any(t.any() for t in zero[1:])


def test_layouts():
    """Heads as a dimension, slices of a fused projection, an expanded context (its gradient summed by expand), broadcast output gradients."""
    dev = torch.device("cuda:0")
    B, N, H, d = 2, 70, 4, 64
    C = H * d
    qkv = randn((B, N, 3 * C), 1, BF16).to(dev)
    dout = randn((B, N, C), 2, BF16, 0.1).to(dev)
    q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    ref = step(q.contiguous(), k.contiguous(), v.contiguous(), H, dout)
    assert all(torch.equal(a, b) for a, b in zip(ref, step(q, k, v, H, dout)))
    four = [t.unflatten(2, (H, d)).transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    got = step(*four, H, dout.unflatten(2, (H, d)).transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(a, b.flatten(2)) for a, b in zip(ref, got))
    leaf = qkv.detach().requires_grad_(True)                                      # one leaf, three slices
    out = ops.cross_attention(leaf[..., :C], leaf[..., C:2 * C], leaf[..., 2 * C:], H)
    whole = torch.autograd.grad(out, leaf, dout)[0]
    assert torch.equal(whole, torch.cat(ref[1:], -1))
    ones = step(q, k, v, H, torch.ones_like(dout))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    assert all(torch.equal(a, b) for a, b in zip(ones[1:], torch.autograd.grad(ops.cross_attention(*leaves, H).sum(), leaves)))
    kl = k[:1].detach().requires_grad_(True)
    dk = torch.autograd.grad(ops.cross_attention(q, kl.expand(B, N, C), v[:1].expand(B, N, C), H), kl, dout)[0]
    assert dk.shape == kl.shape
    for Nk in (70, 200):                                                          # the gradient of the queries alone, of the context alone
        kk, vv = randn((B, Nk, C), 3, BF16).to(dev), randn((B, Nk, C), 4, BF16).to(dev)
        full = step(q, kk, vv, H, dout)
        ql = q.detach().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(ops.cross_attention(ql, kk, vv, H), ql, dout)[0], full[1])
        vl = vv.detach().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(ops.cross_attention(q, kk, vl, H), vl, dout)[0], full[3])
    e = step(q[:0], k[:0], v[:0], H, dout[:0])
    assert e[1].shape == (0, N, C)


@pytest.mark.parametrize("Nk", [9, 150])
def test_against_differences(Nk):
    """Central differences of sum(w * o) in float64 of the definition at the same (rounded) inputs, in random directions."""
    dev = torch.device("cuda:0")
    B, Nq, H, d = 1, 12, 2, 16
    q, w = randn((B, Nq, H * d), 1, F16).to(dev), randn((B, Nq, H * d), 5, F16).to(dev)
    k, v = (randn((B, Nk, H * d), s, F16).to(dev) for s in (2, 3))
    got = step(q, k, v, H, w)[1:]
    at = [t.double().cpu().view(B, -1, H, d).transpose(1, 2) for t in (q, k, v)]
    wd = w.double().cpu().view(B, Nq, H, d).transpose(1, 2)
    loss = lambda a, b, c: float((torch.softmax(a @ b.transpose(2, 3) * d ** -0.5, -1) @ c * wd).sum())      # noqa: E731
    for i in range(3):
        for seed in range(4):
            e = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
            h = 1e-5
            up, down = ([t + s * h * e if j == i else t for j, t in enumerate(at)] for s in (1, -1))
            diff = (loss(*up) - loss(*down)) / (2 * h)
            g = got[i].double().cpu().view(B, -1, H, d).transpose(1, 2)
            # every entry of the gradient is off by at most a few fp16 half steps (2^-11) of the terms it sums; random signs: 16 * 2^-11 of the norm
            assert abs(float((g * e).sum()) - diff) <= 16 * 2.0 ** -11 * float(g.norm() * e.norm()) / g.numel() ** 0.5 * 4 + 1e-6


def test_graph_and_streams():
    dev = torch.device("cuda:0")
    H, d = 4, 64
    for Nk in (77, 300):
        q, k, v, dout = (randn((3, n, H * d), s, F16).to(dev) for n, s in ((500, 1), (Nk, 2), (Nk, 3), (500, 4)))
        lens = torch.tensor([Nk, 5, 0], dtype=torch.int32, device=dev)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        want = step(q, k, v, H, dout, k_lens=lens)
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got += [step(q, k, v, H, dout, k_lens=lens) for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
        del got
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.cross_attention(*leaves, H, k_lens=lens)
            held = (out.detach(), *torch.autograd.grad(out, leaves, dout))
        for seed, n in ((11, (3, Nk, 1)), (12, (0, 0, Nk)), (13, (Nk, Nk, Nk))):
            with torch.no_grad():
                q.copy_(randn(q.shape, seed, F16))
                dout.copy_(randn(dout.shape, seed + 50, F16))
                lens.copy_(torch.tensor(n, dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, step(q, k, v, H, dout, k_lens=lens)))


def test_block_of_the_three_operators():
    """As a transformer block uses them: the entrance norm of a map, attention to a padded prompt with gradients down to the map, the norm's
    parameters and the prompt, then the frames' tokens over an anchor frame's keys.  Gradients against the same block in float64; the tolerance is
    4 half steps of bf16 (norm out, attention out, two rounded gradients) of the largest entry."""
    dev = torch.device("cuda:0")
    B, Hh, W, H, d, L = 3, 10, 12, 5, 64, 77
    C = H * d
    x = randn((B, Hh, W, C), 1, BF16).to(dev).requires_grad_(True)
    gamma = (1 + 0.2 * randn((C,), 2, torch.float32)).to(dev).requires_grad_(True)
    beta = (0.2 * randn((C,), 3, torch.float32)).to(dev).requires_grad_(True)
    k, v = (randn((B, L, C), s, BF16).to(dev).requires_grad_(True) for s in (4, 5))
    lens = torch.tensor([77, 20, 1], dtype=torch.int32, device=dev)
    w = randn((B, Hh * W, C), 6, BF16).to(dev)
    y = ops.groupnorm_act(x, gamma, beta, groups=32, eps=1e-6, act=ops.ACT_NONE).flatten(1, 2)
    out = ops.cross_attention(y, k, v, H, k_lens=lens)
    leaves = (x, gamma, beta, k, v)
    got = torch.autograd.grad(out, leaves, w)
    ref = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    t = ref[0].view(B, Hh * W, 32, C // 32)
    var, mean = torch.var_mean(t, dim=(1, 3), unbiased=False, keepdim=True)
    yr = ((t - mean) / torch.sqrt(var + 1e-6)).view(B, Hh * W, C) * ref[1] + ref[2]
    hs = lambda z: z.view(B, -1, H, d).transpose(1, 2)                                     # noqa: E731
    s = (hs(yr) @ hs(ref[3]).transpose(2, 3) * d ** -0.5).masked_fill(torch.arange(L) >= lens.cpu().view(B, 1, 1, 1), -float("inf"))
    o = (torch.softmax(s, -1) @ hs(ref[4])).transpose(1, 2).reshape(B, Hh * W, C)
    want = torch.autograd.grad(o, ref, w.double().cpu())
    assert (out.detach().double().cpu() - o).abs().max() <= 4 * 2.0 ** -8 * o.abs().max()
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).abs().max() <= 4 * 2.0 ** -8 * b.abs().max(), a.shape
    with torch.no_grad():
        both = ops.prefix_attention(out, out[0], y[0], out, y, H)                          # every frame over the anchor frame's keys and its own
    Reference(out, out, y, H, None, None, None, None, out[0], y[0]).check(both)
