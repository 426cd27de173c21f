"""Edges of the context operators: the causal limit without a prefix, samples and keys that one sample of a shared context lacks, remainders of short contexts,
maps far from zero (bounds: tests/tools_context_attention.py, tests/test_gpu_norm_act.py)."""
import os
import sys

import pytest
import torch

from vidseg_diffusion_amd import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from tools_context_attention import Reference, randn  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,dtype,lens", [
    (1, 64, 64, 1, 1, 64, F16, None),
    (2, 77, 77, 2, 2, 64, BF16, (77, 40)),                   # 40 tokens and 77 queries: the first 37 see nothing
    (3, 70, 96, 4, 2, 64, F16, (96, 70, 0)),
    (2, 32, 77, 4, 1, 96, F16, (77, 5)),                     # 128 rows of a group of four heads
    (2, 64, 96, 2, 2, 96, BF16, (90, 64)),
    (2, 96, 64, 2, 1, 128, F16, (64, 33)),
    (1, 130, 96, 3, 3, 128, BF16, None),
    (2, 5, 9, 26, 2, 40, F16, (9, 2)),                       # 65 rows, all of them groups
    (2, 200, 300, 2, 2, 80, F16, (300, 200)),                # a context over 96 keys
])
def test_causal_without_a_prefix(B, Nq, Nk, H, Hk, d, dtype, lens):
    """The own tokens alone, whatever their number: query i sees keys up to lens - Nq + i."""
    dev = torch.device("cuda:0")
    q = randn((B, Nq, H * d), 1, dtype, 1.5).to(dev)
    k, v = (randn((B, Nk, Hk * d), s, dtype).to(dev) for s in (2, 3))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    none = k[0, :0]
    out, lse = ops.prefix_attention(q, none, none, k, v, H, kv_heads=Hk, k_lens=n, causal=True, return_lse=True)
    Reference(q, k, v, H, Hk, n, causal=True).check(out, lse)
    free, f_lse = ops.prefix_attention(q, none, none, k, v, H, kv_heads=Hk, k_lens=n, return_lse=True)
    Reference(q, k, v, H, Hk, n).check(free, f_lse)


def step(q, k, v, heads, dout, **how):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, heads, **how)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk,d", [(70, 77, 64), (1, 77, 64), (70, 300, 64), (700, 300, 128), (70, 100, 80)])
def test_samples_without_a_key_beside_a_shared_context(Nq, Nk, d, dtype):
    """One context for the batch; the samples without a key hold NaN or infinities in their queries and in the gradients of their rows: no gradient of
    the context and of the other samples changes, theirs are zero."""
    dev = torch.device("cuda:0")
    q, dout = randn((4, Nq, 2 * d), 1, dtype).to(dev), randn((4, Nq, 2 * d), 4, dtype).to(dev)
    k, v = (randn((1, Nk, 2 * d), s, dtype).to(dev) for s in (2, 3))
    lens = torch.tensor([Nk, 0, 5, 0], dtype=torch.int32, device=dev)
    mask = torch.arange(Nk, device=dev) < lens.view(4, 1)
    for how in (dict(k_lens=lens), dict(key_mask=mask)):
        want = step(q, k, v, 2, dout, **how)
        Reference(q, k, v, 2, None, lens).check_gradients(dout, *want[1:], True)
        for bad in (float("nan"), float("inf")):
            q2, g2 = q.clone(), dout.clone()
            q2[1], g2[1], q2[3] = bad, bad, bad
            for a, b in zip(want, step(q2, k, v, 2, g2, **how)):
                assert torch.equal(a, b)
        assert not want[1][[1, 3]].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk", [(70, 77), (1, 77), (70, 300), (1, 300)])
def test_gradients_of_rows_without_a_key(Nq, Nk, dtype):
    """A padded sample's rows carry NaN or infinities in the output's gradient: its own gradients are zero, the others' unchanged."""
    dev = torch.device("cuda:0")
    q, k, v, dout = (randn((3, n, 128), s, dtype).to(dev) for n, s in ((Nq, 1), (Nk, 2), (Nk, 3), (Nq, 4)))
    lens = torch.tensor([Nk, 0, 5], dtype=torch.int32, device=dev)
    mask = torch.arange(Nk, device=dev) < lens.view(3, 1)
    for how in (dict(k_lens=lens), dict(key_mask=mask)):
        want = step(q, k, v, 2, dout, **how)
        for bad in (float("nan"), float("inf")):
            q2, g2 = q.clone(), dout.clone()
            q2[1], g2[1] = bad, bad
            for a, b in zip(want, step(q2, k, v, 2, g2, **how)):
                assert torch.equal(a, b)
        assert not any(t[1].any() for t in want[1:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk,d", [(70, 77, 64), (1, 77, 64), (70, 128, 128), (70, 300, 64)])
def test_keys_that_one_sample_of_a_shared_context_lacks(Nq, Nk, d, dtype):
    """Keys that exist for the first sample only hold NaN or infinities: nothing of that reaches the second sample's result and gradient."""
    dev = torch.device("cuda:0")
    q, dout = randn((3, Nq, 2 * d), 1, dtype).to(dev), randn((3, Nq, 2 * d), 4, dtype).to(dev)
    k, v = (randn((1, Nk, 2 * d), s, dtype).to(dev) for s in (2, 3))
    lens = torch.tensor([30, Nk, 30], dtype=torch.int32, device=dev)
    mask = torch.arange(Nk, device=dev) < lens.view(3, 1)
    for how in (dict(k_lens=lens), dict(key_mask=mask)):
        want = step(q, k, v, 2, dout, **how)
        Reference(q, k, v, 2, None, lens).check_gradients(dout, *want[1:], True)
        for bad in (float("nan"), float("inf")):
            for which in (0, 1):
                kv = [k.clone(), v.clone()]
                kv[which][:, 30:] = bad
                got = step(q, *kv, 2, dout, **how)
                for b in (0, 2):
                    assert torch.equal(got[0][b], want[0][b]) and torch.equal(got[1][b], want[1][b])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Nq,Nk,lens", [(100, 77, (77, 3)), (100, 96, (0, 96)), (3, 77, (77, 5)), (100, 300, (300, 1)), (2, 2600, (2600, 0))])
def test_what_the_rounding_left(Nq, Nk, lens, dtype):
    """The C entry's out_lo at every length: written everywhere, at most half a step of out, and not zero where several keys were averaged."""
    from vidseg_diffusion_amd import _lib
    dev = torch.device("cuda:0")
    B, H, d = 2, 2, 64
    q = randn((B, Nq, H, d), 1, dtype, 1.5).to(dev)
    k, v = (randn((B, Nk, H, d), s, dtype).to(dev) for s in (2, 3))
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    out, left = torch.full_like(q, float("nan")), torch.full_like(q, float("nan"))
    kib = _lib.lib().vidseg_context_attention_scratch_kib(B, Nq, 0, Nk, H, H, d)
    scratch = torch.empty(max(kib, 1) * 256, device=dev)
    own = [a for t in (k, v) for a in (t.data_ptr(), *t.stride()[:3])]
    _lib.call("vidseg_context_attention_fwd", q.data_ptr(), *q.stride()[:3], *(None, 0, 0) * 2, *own, n.data_ptr(), None, 0, out.data_ptr(), left.data_ptr(), None,
              1 if dtype == F16 else 2, B, Nq, 0, Nk, H, H, d, d ** -0.5, 0, scratch.data_ptr(), kib, torch.cuda.current_stream().cuda_stream)
    Reference(q.flatten(2), k.flatten(2), v.flatten(2), H, None, n).check(out.flatten(2))
    assert torch.isfinite(left).all()
    half = torch.finfo(dtype).eps / 2
    # what the rounding left is at most half a step of out (half a subnormal step of fp16 at the least)
    assert (left.double().abs() <= half * out.double().abs() * (1 + 2 * half) + 2.0 ** -25).all()
    if max(lens) > 1:
        assert (left != 0).float().mean() > 0.2 * sum(x > 0 for x in lens) / 2


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("B,dims,C,groups", [(2, (8, 8), 1280, 32), (1, (1,), 64, 8), (2, (33, 7), 640, 32), (2, (2000,), 30, 3), (1, (700,), 2560, 32)])
def test_maps_far_from_zero(B, dims, C, groups, dtype):
    """Means whose square passes fp32's range, spreads whose square does not."""
    from test_gpu_norm_act import check_all, data
    dev = torch.device("cuda:0")
    for far in (3e19, -1e25):
        x, gamma, beta, dy = data(B, dims, C, torch.float32, 5, dev)
        x = (far + x * 2.0 ** 58).to(dtype)                  # bf16: steps of 2^57 at 3e19; at 1e25 (steps of 2^75) mostly one value, some beside it
        check_all(x, gamma, beta, dy.to(dtype), groups, True)
    x = torch.full((B, *dims, C), 3e38, device=dev, dtype=dtype)
    beta = torch.linspace(-1, 1, C, device=dev)
    y = ops.groupnorm_act(x, torch.ones(C, device=dev), beta, groups=groups, act=ops.ACT_NONE)
    assert torch.equal(y, beta.to(dtype).expand_as(y))


@pytest.mark.parametrize("eps", [0.0, 1e-20, 1e-17])
def test_small_spreads_without_an_eps(eps):
    """Deviations of 2^-60, whose squares are the variance where eps is zero and nothing beside it where eps is not; ordinary maps on both sides of 2^-60."""
    from test_gpu_norm_act import check_all, data
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(2, (33, 7), 640, torch.float32, 5, dev)
    check_all(x, gamma, beta, dy, 32, True, eps)
    check_all(x * 2.0 ** -60, gamma, beta, dy, 32, False, eps)


@pytest.mark.parametrize("Nk", [77, 300])
def test_captured_calls_on_one_context(Nk):
    """One context for the batch, forward and gradients captured once and replayed with other lengths, samples without a key among them; beside it a causal call
    without a prefix."""
    dev = torch.device("cuda:0")
    B, Nq, H = 4, 150, 2
    q, dout = (randn((B, Nq, H * 64), s, F16).to(dev) for s in (1, 4))
    k, v = (randn((1, Nk, H * 64), s, F16).to(dev) for s in (2, 3))
    own = k.expand(B, Nk, H * 64)
    lens = torch.tensor([Nk, 0, 5, 9], dtype=torch.int32, device=dev)

    def calls(leaves):
        out = ops.cross_attention(*leaves, H, k_lens=lens)
        with torch.no_grad():
            late = ops.prefix_attention(q, own[0, :0], own[0, :0], own, own, H, k_lens=lens, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout), late)
    fresh = lambda: [t.detach().clone().requires_grad_(True) for t in (q, k, v)]               # noqa: E731
    calls(fresh())
    leaves = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls(leaves)
    for seed, n in ((11, (0, Nk, 0, 3)), (12, (0, 0, 0, Nk)), (13, (Nk, Nk, Nk, Nk)), (14, (0, 0, 0, 0))):
        with torch.no_grad():
            q.copy_(randn(q.shape, seed, F16))
            leaves[0].copy_(q)
            lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = calls(fresh())
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        Reference(q, k, v, H, None, lens).check_gradients(dout, *want[1:4], True)
        Reference(q, own, own, H, None, lens, causal=True).check(want[4])
