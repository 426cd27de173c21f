"""ops.cross_attention and ops.prefix_attention against float64, forward (bounds: tests/tools_context_attention.py)."""
import os
import sys

import pytest
import torch

from vidseg_diffusion_amd import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from tools_context_attention import Reference, randn  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

CROSS = [  # B, Nq, Nk, H, Hk, d, dtype, lens, shared context
    (2, 64, 77, 5, 5, 64, F16, None, False),
    (3, 130, 77, 2, 2, 64, BF16, (77, 1, 0), False),           # a sample without a key
    (1, 1, 1, 1, 1, 8, F16, None, False),                      # the smallest call
    (2, 1, 257, 16, 16, 80, BF16, (257, 100), False),          # one query: waves split the keys
    (4, 1, 2500, 8, 2, 128, F16, (2500, 0, 33, 1024), False),  # one query, long keys: several blocks a row, joined
    (2, 31, 65, 4, 1, 40, BF16, (64, 65), False),              # a group of 4 heads: 124 rows on one key head
    (2, 33, 200, 3, 3, 96, F16, (129, 200), True),             # one context for the batch, its length by sample
    (1, 5, 300, 6, 2, 104, BF16, (300,), False),
    (2, 257, 129, 4, 2, 128, F16, (128, 129), False),
    (1, 700, 1031, 1, 1, 24, F16, None, False),                # few row tiles, keys over several blocks
    (1, 128, 64, 2, 2, 64, BF16, None, False),                 # exact tiles
    (2, 40, 0, 2, 2, 64, F16, None, False),                    # no keys at all
    (9, 3, 64, 8, 8, 16, F16, (64, 63, 33, 32, 31, 1, 0, 64, 5), False),
    (2, 130, 96, 3, 3, 80, F16, (96, 81), False),                     # around the longest context that one block holds
    (2, 130, 97, 3, 3, 128, BF16, (97, 96), False),
    (3, 70, 85, 6, 2, 40, F16, (85, 16, 17), True),
]


@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,dtype,lens,shared", CROSS)
def test_cross_attention(B, Nq, Nk, H, Hk, d, dtype, lens, shared):
    dev = torch.device("cuda:0")
    q = randn((B, Nq, H * d), 1, dtype, 1.5).to(dev)
    k, v = (randn((1 if shared else B, Nk, Hk * d), s, dtype).to(dev) for s in (2, 3))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = ops.cross_attention(q, k, v, H, kv_heads=Hk, k_lens=n, return_lse=True)
    assert out.shape == q.shape and out.dtype == dtype and lse.shape == (B, H, Nq)
    ref = Reference(q, k, v, H, Hk, n)
    ref.check(out, lse)
    if lens is not None:
        empty = torch.tensor(lens, device=dev) == 0
        assert not out[empty].any()
    assert torch.equal(out, ops.cross_attention(q, k, v, H, kv_heads=Hk, k_lens=n))


PREFIX = [  # B, Nq, Np, Nk, H, Hk, d, dtype, lens, causal
    (4, 1, 77, 33, 16, 16, 64, F16, (33, 1, 7, 20), True),
    (5, 1, 1000, 65, 8, 2, 128, BF16, (65, 64, 1, 0, 33), False),     # a sample with the prefix alone
    (3, 4, 130, 40, 4, 1, 80, F16, (40, 4, 17), True),                # several new tokens
    (2, 3, 10, 9, 2, 2, 64, F16, (2, 9), True),                       # more queries than own keys: the first see the prefix only
    (2, 3, 0, 9, 2, 2, 64, BF16, (2, 9), True),                       # ... and without a prefix nothing
    (2, 200, 129, 70, 3, 3, 64, F16, None, False),                    # many rows: prefix and own keys in one pass
    (2, 150, 64, 150, 2, 1, 96, BF16, (150, 149), True),
    (40, 2, 300, 20, 4, 2, 64, F16, None, True),                      # stacked rows of many samples
    (2, 50, 64, 0, 2, 2, 64, F16, None, False),                       # no own keys
    (1, 1, 5000, 3, 1, 1, 64, BF16, (3,), True),                      # one row, one long prefix
    (3, 40, 90, 64, 2, 2, 48, F16, (0, 64, 10), False),
    (40, 2, 600, 20, 4, 2, 64, BF16, None, True),                     # stacked rows of many samples, few rows of their own
    (64, 1, 1000, 40, 8, 2, 128, F16, None, True),
    (3, 40, 700, 64, 2, 2, 48, F16, (0, 64, 10), False),              # stacked rows, and more than 32 of their own
    (2, 1, 2600, 33, 4, 4, 80, BF16, (33, 2), True),                  # few rows in all, the prefix dealt out over blocks
    (1, 1, 5000, 2100, 2, 2, 64, F16, (2050,), True),                 # one sample: prefix and own keys in one walk
    (70, 2, 500, 20, 4, 2, 64, BF16, None, True),                     # a prefix long enough to stack the rows: own rows few,
    (3, 40, 11000, 64, 2, 2, 48, F16, (0, 64, 10), False),            # own rows many,
    (2, 1, 17000, 33, 4, 4, 80, BF16, (33, 2), True),                 # few rows in all,
    (45, 1, 900, 0, 6, 2, 104, F16, None, False),                     # no own keys
]


@pytest.mark.parametrize("B,Nq,Np,Nk,H,Hk,d,dtype,lens,causal", PREFIX)
def test_prefix_attention(B, Nq, Np, Nk, H, Hk, d, dtype, lens, causal):
    dev = torch.device("cuda:0")
    q = randn((B, Nq, H * d), 1, dtype, 1.5).to(dev)
    k, v = (randn((B, Nk, Hk * d), s, dtype).to(dev) for s in (2, 3))
    kp, vp = (randn((Np, Hk * d), s, dtype).to(dev) for s in (4, 5))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = ops.prefix_attention(q, kp, vp, k, v, H, kv_heads=Hk, k_lens=n, causal=causal, return_lse=True)
    Reference(q, k, v, H, Hk, n, None, None, kp, vp, causal).check(out, lse)
    assert torch.equal(out, ops.prefix_attention(q, kp, vp, k, v, H, kv_heads=Hk, k_lens=n, causal=causal))


@pytest.mark.parametrize("Nq,d,dtype", [(70, 64, F16), (1, 64, BF16), (33, 128, BF16), (200, 80, F16)])
def test_key_mask_and_poison(Nq, d, dtype):
    """A mask that empties whole tiles and one sample; NaN and infinities in every place that does not exist change no bit."""
    dev = torch.device("cuda:0")
    B, Nk, H = 3, 330, 2
    q = randn((B, Nq, H * d), 1, dtype).to(dev)
    k, v = (randn((B, Nk, H * d), s, dtype).to(dev) for s in (2, 3))
    g = torch.Generator().manual_seed(4)
    mask = torch.rand((B, Nk), generator=g) < 0.5
    mask[0, 64:192] = False
    mask[1] = False
    mask = mask.to(dev)
    lens = torch.tensor([330, 330, 201], dtype=torch.int32, device=dev)
    out, lse = ops.cross_attention(q, k, v, H, k_lens=lens, key_mask=mask, return_lse=True)
    Reference(q, k, v, H, None, lens, mask).check(out, lse)
    assert not out[1].any()
    dead = ~(mask & (torch.arange(Nk, device=dev) < lens.view(B, 1)))
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        k2, v2 = (t.masked_fill(dead.unsqueeze(-1), bad) for t in (k, v))
        o2, l2 = ops.cross_attention(q, k2, v2, H, k_lens=lens, key_mask=mask, return_lse=True)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
    one = ops.cross_attention(q, k, v, H, key_mask=mask[:1])                  # one mask for all samples
    Reference(q, k, v, H, None, None, mask[:1].expand(B, Nk)).check(one)


@pytest.mark.parametrize("Nq,Nk", [(70, 77), (1, 77), (70, 300), (1, 300)])
def test_nothing_to_attend_to_and_no_number_to_ask_with(Nq, Nk):
    """A padded sample: no key, and queries that hold NaN and infinities.  Zeros, log-sum-exp -inf, gradients of zero, and no other sample's values change."""
    dev = torch.device("cuda:0")
    q, k, v, w = (randn((3, n, 128), s, F16).to(dev) for n, s in ((Nq, 1), (Nk, 2), (Nk, 3), (Nq, 4)))
    lens = torch.tensor([Nk, 0, 5], dtype=torch.int32, device=dev)

    def step(q):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out, lse = ops.cross_attention(*leaves, 2, k_lens=lens, return_lse=True)
        return (out.detach(), lse, *torch.autograd.grad(out, leaves, w))
    want = step(q)
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[1] = bad
        for a, b in zip(want, step(q2)):
            assert torch.equal(a, b)
        mask = torch.arange(Nk, device=dev) < lens.view(3, 1)
        assert torch.equal(want[0], ops.cross_attention(q2, k, v, 2, key_mask=mask))
        assert torch.equal(want[0], ops.prefix_attention(q2, k[0, :0], v[0, :0], k, v, 2, k_lens=lens))
    assert not want[0][1].any() and torch.isneginf(want[1][1]).all() and not any(t[1].any() for t in want[2:])


def test_layouts_and_strides():
    """Column slices of a fused projection, heads as a dimension in either order, a context expanded over the batch, unaligned views (copied)."""
    dev = torch.device("cuda:0")
    B, N, H, d = 2, 70, 4, 64
    C = H * d
    qkv = randn((B, N, 3 * C), 1, F16).to(dev)
    q, k, v = qkv[..., :C], qkv[..., C:2 * C], qkv[..., 2 * C:]
    ref = ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), H)
    assert torch.equal(ops.cross_attention(q, k, v, H), ref)
    r4 = ref.view(B, N, H, d)
    q4, k4, v4 = (t.unflatten(2, (H, d)) for t in (q, k, v))
    assert torch.equal(ops.cross_attention(q4, k4, v4, H), r4)
    bhnd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q4, k4, v4)]
    assert torch.equal(ops.cross_attention(*bhnd, H), r4)
    shifted = torch.empty(B * N * C + 1, dtype=F16, device=dev)[1:].view(B, N, C).copy_(k)
    assert torch.equal(ops.cross_attention(q, shifted, v, H), ref)
    ctx_k, ctx_v = k[:1], v[:1]
    assert torch.equal(ops.cross_attention(q, ctx_k, ctx_v, H), ops.cross_attention(q, ctx_k.expand(B, N, C), ctx_v.expand(B, N, C), H))
    pre = ops.prefix_attention(q, k[0], v[0], k, v, H)
    assert torch.equal(pre, ops.prefix_attention(q4, k4[0], v4[0], k4, v4, H).flatten(2))
    assert ops.cross_attention(q[:0], k[:0], v[:0], H).shape == (0, N, C) and ops.cross_attention(q[:, :0], k, v, H).shape == (B, 0, C)


def test_extreme_scores():
    """Scores up to several thousand in both directions: the running maximum moves by more than exp2's range between tiles."""
    dev = torch.device("cuda:0")
    for dtype in (F16, BF16):
        for Nq in (1, 150):
            q = randn((1, Nq, 64), 1, dtype, 30.0).to(dev)
            k = (randn((1, 400, 64), 2, dtype, 30.0) * torch.linspace(0.01, 1, 400).view(1, 400, 1).to(dtype)).to(dev)
            v = randn((1, 400, 64), 3, dtype).to(dev)
            out, lse = ops.cross_attention(q, k, v, 1, return_lse=True)
            Reference(q, k, v, 1).check(out, lse)


def test_prefix_equals_one_context():
    """The prefix and the own keys side by side are one softmax: equal within the bounds to cross attention over their concatenation."""
    dev = torch.device("cuda:0")
    B, H, d = 6, 4, 64
    for Nq in (1, 20, 150):
        q = randn((B, Nq, H * d), 1, BF16).to(dev)
        k, v = (randn((B, 50, H * d), s, BF16).to(dev) for s in (2, 3))
        kp, vp = (randn((200, H * d), s, BF16).to(dev) for s in (4, 5))
        a = ops.prefix_attention(q, kp, vp, k, v, H)
        b = ops.cross_attention(q, torch.cat([kp.expand(B, -1, -1), k], 1), torch.cat([vp.expand(B, -1, -1), v], 1), H)
        ref = Reference(q, k, v, H, None, None, None, None, kp, vp)
        ref.check(a)
        ref.check(b)


def test_offsets_beyond_32_bits():
    """Own keys of the last sample start more than 2^32 elements behind the first (a strided cache), and the last prefix row likewise."""
    dev = torch.device("cuda:0")
    d = 64
    rows = (1 << 32) // d + 1000
    cache = torch.empty((rows, d), dtype=F16, device=dev)                       # 8.6 GB
    k = cache.as_strided((2, 80, d), ((rows - 100) * d, d, 1))
    k.copy_(randn((2, 80, d), 2, F16).to(dev))
    q, v = randn((2, 3, d), 1, F16).to(dev), randn((2, 80, d), 3, F16).to(dev)
    Reference(q, k, v, 1).check(ops.cross_attention(q, k, v, 1))
    kp = cache.as_strided((3, d), ((rows - 200) // 2 * d, 1))
    kp.copy_(randn((3, d), 4, F16).to(dev))
    vp = randn((3, d), 5, F16).to(dev)
    Reference(q, v, v, 1, None, None, None, None, kp, vp).check(ops.prefix_attention(q, kp, vp, v, v, 1))


def test_streams_and_graph():
    dev = torch.device("cuda:0")
    B, H, d = 4, 8, 64
    q, k, v = (randn((B, n, H * d), s, F16).to(dev) for n, s in ((1, 1), (900, 2), (900, 3)))
    kp, vp = (randn((700, H * d), s, F16).to(dev) for s in (4, 5))
    lens = torch.tensor([900, 1, 0, 333], dtype=torch.int32, device=dev)
    ref = ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens), ops.cross_attention(q, k, v, H, k_lens=lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                                           # two calls at once: no scratch between them
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(10):
                got.append((ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens), ops.cross_attention(q, k, v, H, k_lens=lens)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, ref))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens), ops.cross_attention(q, k, v, H, k_lens=lens)))
        graphs.append(g)
    for seed, n in ((11, (5, 900, 64, 128)), (12, (0, 0, 1, 900)), (13, (900, 900, 900, 900))):
        q.copy_(randn(q.shape, seed, F16))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens), ops.cross_attention(q, k, v, H, k_lens=lens)
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_graphs_of_stacked_rows():
    """Single tokens of many samples behind a prefix long enough to be dealt out and joined: two captured graphs in flight on two streams, each with its own scratch."""
    dev = torch.device("cuda:0")
    B, H, d = 40, 4, 64
    q, k, v = (randn((B, n, H * d), s, BF16).to(dev) for n, s in ((1, 1), (70, 2), (70, 3)))
    kp, vp = (randn((3000, H * d), s, BF16).to(dev) for s in (4, 5))
    lens = torch.full((B,), 70, dtype=torch.int32, device=dev)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens, causal=True))
        graphs.append(g)
    for seed in (11, 12, 13):
        q.copy_(randn(q.shape, seed, BF16))
        lens.copy_(torch.randint(0, 71, (B,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = ops.prefix_attention(q, kp, vp, k, v, H, k_lens=lens, causal=True)
        assert all(torch.equal(o, want) for o in outs)
        Reference(q, k, v, H, None, lens, None, None, kp, vp, True).check(want)
