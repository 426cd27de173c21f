"""Every variant of the context attention kernels that a call can reach, in both types: the short, tiled, few-row and stacked forms and both forms of the gradients
at each padded head width (bounds: tests/tools_context_attention.py)."""
import os
import sys

import pytest
import torch

from vidseg_diffusion_amd import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from tools_context_attention import Reference, randn  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def tensors(B, Nq, Nk, H, Hk, d, dtype, lens, Np=0):
    dev = torch.device("cuda:0")
    q = randn((B, Nq, H * d), 1, dtype, 1.5).to(dev)
    k, v = (randn((B, Nk, Hk * d), s, dtype).to(dev) for s in (2, 3))
    kp, vp = (randn((Np, Hk * d), s, dtype).to(dev) for s in (4, 5))
    return q, k, v, kp, vp, None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,d,lens", [
    (2, 70, 77, 2, 2, 128, (77, 16)),
    (3, 130, 96, 4, 2, 104, (96, 81, 0)),                     # groups, a width below the padded one, half blocks of 16 keys
    (1, 2100, 33, 1, 1, 112, None),                           # several tiles a wave
    (2, 64, 1, 2, 2, 128, (1, 0)),
    (2, 515, 80, 3, 1, 120, (80, 47)),
    (2, 99, 96, 2, 2, 96, (96, 33)),
    (2, 99, 49, 2, 2, 64, (49, 48)),
])
def test_short_contexts(B, Nq, Nk, H, Hk, d, lens, dtype):
    q, k, v, _, _, n = tensors(B, Nq, Nk, H, Hk, d, dtype, lens)
    out, lse = ops.cross_attention(q, k, v, H, kv_heads=Hk, k_lens=n, return_lse=True)
    Reference(q, k, v, H, Hk, n).check(out, lse)
    g = torch.Generator().manual_seed(4)
    mask = (torch.rand((B, Nk), generator=g) < 0.5).to(q.device)
    out = ops.cross_attention(q, k, v, H, kv_heads=Hk, k_lens=n, key_mask=mask)
    Reference(q, k, v, H, Hk, n, mask).check(out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 40, 96, 72, 128, 104])
@pytest.mark.parametrize("B,Nq,Np,Nk,H,Hk,lens", [
    (70, 2, 500, 20, 4, 2, None),                             # stacked rows for the prefix, few rows of their own
    (2, 1, 17000, 33, 4, 4, (33, 2)),                         # few rows in all
    (3, 40, 11000, 64, 2, 2, (40, 64, 10)),                   # stacked rows, own rows many
    (2, 130, 100, 200, 4, 2, (200, 131)),                     # prefix and own keys in one walk
])
def test_shared_prefix(B, Nq, Np, Nk, H, Hk, lens, d, dtype):
    q, k, v, kp, vp, n = tensors(B, Nq, Nk, H, Hk, d, dtype, lens, Np)
    for causal in (True, False):
        out, lse = ops.prefix_attention(q, kp, vp, k, v, H, kv_heads=Hk, k_lens=n, causal=causal, return_lse=True)
        Reference(q, k, v, H, Hk, n, None, None, kp, vp, causal).check(out, lse, f"causal={causal}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Nq,Np,Nk,H,Hk,d,lens", [
    (2, 300, 70, 300, 2, 2, 64, (300, 180)),                  # a prompt behind a prefix: more queries than own keys in use
    (1, 515, 129, 515, 4, 1, 64, None),
    (2, 257, 64, 400, 2, 1, 128, (400, 257)),
    (2, 200, 1, 200, 3, 3, 80, (200, 1)),
    (3, 130, 0, 130, 2, 2, 128, (130, 64, 0)),
])
def test_causal_prompts(B, Nq, Np, Nk, H, Hk, d, lens, dtype):
    q, k, v, kp, vp, n = tensors(B, Nq, Nk, H, Hk, d, dtype, lens, Np)
    out, lse = ops.prefix_attention(q, kp, vp, k, v, H, kv_heads=Hk, k_lens=n, causal=True, return_lse=True)
    Reference(q, k, v, H, Hk, n, None, None, kp, vp, True).check(out, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 80, 128, 104])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,lens,shared", [
    (2, 130, 100, 4, 2, (100, 33), False),                    # one pass for all three gradients
    (3, 70, 128, 2, 2, (128, 0, 65), True),
    (2, 130, 270, 4, 2, (270, 129), False),                   # two passes
    (3, 70, 150, 2, 2, (150, 0, 140), True),
    (1, 1500, 60, 1, 1, None, False),                         # partial sums joined
    (1, 1500, 140, 1, 1, None, False),
])
def test_gradients(B, Nq, Nk, H, Hk, lens, shared, d, dtype):
    q, k, v, _, _, n = tensors(B, Nq, Nk, H, Hk, d, dtype, lens)
    if shared:
        k, v = k[:1], v[:1]
    dout = randn(q.shape, 6, dtype, 0.1).to(q.device)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, H, kv_heads=Hk, k_lens=n)
    got = torch.autograd.grad(out, leaves, dout)
    ref = Reference(q, k, v, H, Hk, n)
    ref.check(out.detach())
    ref.check_gradients(dout, *got, shared)
