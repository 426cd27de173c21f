"""ops.groupnorm_act against a float64 evaluation of the same formula, forward and gradients.

Tolerances: the result is rounded once, at most half a step (finfo.eps / 2 relative); what is computed before it is fp32, whose error is
counted in units u = 2^-24 of the largest term that enters:
  y:      z = (x - mean) rstd gamma + beta; each operand carries a few u, the largest terms are |x| rstd |gamma| and |beta|  ->  16 u of their sum
          (SiLU's slope is at most 1.1 and exp2 / rcp are good to a few u)
  dx:     rstd (gamma dz - a - xh b), |a| <= max|gamma dz|, |b| <= max|gamma dz xh|                                         ->  64 u rstd max|gamma dz| (2 + max|xh|^2)
          plus the error of xh itself (above) times dz's slope
  dgamma, dbeta: sums in a fixed order whose chains are at most rows per lane + lanes + chunks + samples < 1024 long     ->  1024 u sum|terms|
"""
import pytest
import torch

from vidseg_diffusion_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, gamma, beta, groups, eps, silu, dy=None):
    """float64 on the CPU; x [B, HW, C]."""
    x, gamma, beta = (t.detach().double().cpu() for t in (x, gamma, beta))
    B, HW, C = x.shape
    t = x.view(B, HW, groups, C // groups)
    mean = t.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((t - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xh = ((t - mean) * rstd).view(B, HW, C)
    z = xh * gamma + beta
    sig = torch.sigmoid(z)
    y = z * sig if silu else z
    if dy is None:
        return y, xh, rstd
    dy = dy.double().cpu()
    dz = dy * (sig * (1 + z * (1 - sig))) if silu else dy
    g = (dz * gamma).view(B, HW, groups, -1)
    h = xh.view(B, HW, groups, -1)
    dx = rstd * (g - g.mean((1, 3), keepdim=True) - h * (g * h).mean((1, 3), keepdim=True))
    return y, dx.view(B, HW, C), (dz * xh).sum((0, 1)), dz.sum((0, 1)), xh, rstd, dz


def inside(got, ref, slack, what):
    got = got.detach().double().cpu()
    tol = torch.finfo(what[0]).eps / 2 * ref.abs() + slack
    if what[0] == torch.float16:
        tol = tol + 2.0 ** -25                                       # half a step of fp16's subnormals
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{what[1]}: {int(bad.sum())} of {bad.numel()} outside, worst {((got - ref).abs() / tol.clamp_min(1e-300)).max():.3g} of the tolerance"


CASES = [  # B, HW dims, C, groups, silu, dtype
    (2, (8, 8), 1280, 32, True, torch.float32),
    (3, (16, 16), 320, 32, True, torch.float16),              # groups of 10 channels end inside 16-byte pieces
    (2, (33, 7), 640, 32, False, torch.bfloat16),
    (1, (1,), 64, 8, True, torch.float32),                    # one row
    (1, (1,), 8, 8, True, torch.float16),                     # one value per group: z = beta
    (5, (3,), 36, 4, True, torch.float16),                    # rows of 72 bytes: single-value accesses
    (2, (129,), 30, 3, False, torch.bfloat16),
    (2, (50, 41), 24, 1, True, torch.float32),                # one group
    (1, (700,), 2560, 32, True, torch.bfloat16),              # more 16-byte columns than threads
    (1, (20,), 8192, 32, True, torch.float32),                # the widest map
    (1, (20,), 8191, 1, True, torch.float32),
    (28, (64, 64), 320, 32, True, torch.float16),
]


def data(B, dims, C, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, *dims, C), generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + torch.randn(C, generator=g)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    dy = 0.1 * torch.randn((B, *dims, C), generator=g)
    return x.to(dtype).to(dev), gamma.to(dev), beta.to(dev), dy.to(dtype).to(dev)


def check_all(x, gamma, beta, dy, groups, silu, eps=1e-5):
    C = x.shape[-1]
    B = x.shape[0]
    leaves = [t.detach().requires_grad_(True) for t in (x, gamma, beta)]
    y = ops.groupnorm_act(*leaves, groups=groups, eps=eps, act=ops.ACT_SILU if silu else ops.ACT_NONE)
    plain = ops.groupnorm_act(x.detach(), gamma, beta, groups=groups, eps=eps, act=ops.ACT_SILU if silu else ops.ACT_NONE)
    assert torch.equal(y, plain) and y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    dx, dg, db = torch.autograd.grad(y, leaves, dy)
    ry, rdx, rdg, rdb, xh, rstd, dz = reference(x.reshape(B, -1, C), gamma, beta, groups, eps, silu, dy.reshape(B, -1, C))
    gmax = gamma.abs().max().double().cpu()
    xs = (x.detach().double().cpu().abs().max() * rstd.max() * gmax + beta.abs().max().double().cpu())
    inside(y.reshape(B, -1, C), ry, 16 * U * xs, (x.dtype, "y"))
    dzm, xm = dz.abs().max(), xh.abs().max()
    slack = 64 * U * rstd.max() * gmax * dzm * (2 + xm ** 2) + (16 * U * xs) * rstd.max() * gmax * dy.abs().max().double().cpu() * (2 + xm) if dy.numel() else 0
    inside(dx.reshape(B, -1, C), rdx, slack, (x.dtype, "dx"))
    # each term of the sums also carries xh's error (16 u of the same terms) times |dy|
    per = (16 * U * xs) * dy.detach().double().cpu().abs().reshape(-1, C).sum(0) * (1 + xm)
    inside(dg, rdg, 1024 * U * (dz * xh).abs().sum((0, 1)) + per, (torch.float32, "dgamma"))
    inside(db, rdb, 1024 * U * dz.abs().sum((0, 1)) + per, (torch.float32, "dbeta"))
    return y, dx, dg, db


@pytest.mark.parametrize("B,dims,C,groups,silu,dtype", CASES)
def test_groupnorm_act(B, dims, C, groups, silu, dtype):
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(B, dims, C, dtype, 11, dev)
    check_all(x, gamma, beta, dy, groups, silu)


def test_far_mean_keeps_its_variance():
    """fp32 values around 4096 with a spread of 1: sums of squares would leave the variance 2^-24 * 4096^2 = 1 wrong."""
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(2, (40, 25), 64, torch.float32, 5, dev)
    check_all(x + 4096.0, gamma, beta, dy, 8, True)


@pytest.mark.parametrize("rows,C,groups,dims", [(1, 8, 8, (20000,)), (1, 320, 32, (64, 64)), (1250, 8, 8, (20000,)), (3, 1280, 32, (40, 40))])
def test_first_rows_far_from_the_others(rows, C, groups, dims):
    """The first rows (of a thread, a chunk, a map) are no good reference for the others: 10^4 away from them."""
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(2, dims, C, torch.float32, 7, dev)
    x.view(2, -1, C)[:, :rows] += 1e4
    check_all(x, gamma, beta, dy, groups, True)


def test_constant_map():
    dev = torch.device("cuda:0")
    x = torch.full((2, 9, 64), 3.0, device=dev)
    gamma, beta = torch.ones(64, device=dev), torch.linspace(-1, 1, 64, device=dev)
    y = ops.groupnorm_act(x, gamma, beta, groups=8, act=ops.ACT_NONE)
    assert torch.equal(y, beta.expand_as(y))                          # a thread's first value is the shift: every difference is exactly zero


def test_slices_and_other_orders():
    """Column slices (a row stride), a sliced batch, a transposed map (copied) and transposed / broadcast gradients."""
    dev = torch.device("cuda:0")
    wide, gamma, beta, dy = data(4, (12, 10), 128, torch.float16, 3, dev)
    g, b = gamma[:64].clone(), beta[:64].clone()
    d = dy[..., :64].clone()
    ref = ops.groupnorm_act(wide[..., 64:].contiguous(), g, b, groups=8)
    for view, dv in ((wide[..., 64:], d), (wide[..., 64:].transpose(1, 2).contiguous().transpose(1, 2), d.transpose(1, 2).contiguous().transpose(1, 2))):
        leaf = view.detach().requires_grad_(True)
        y = ops.groupnorm_act(leaf, g, b, groups=8)
        assert torch.equal(y, ref)
        check_all(view, g, b, dv, 8, True)
    assert torch.equal(ops.groupnorm_act(wide[::2, :, :, 1:65], g, b, groups=8), ops.groupnorm_act(wide[::2, :, :, 1:65].contiguous(), g, b, groups=8))
    leaf = wide[..., :64].detach().requires_grad_(True)
    one = torch.autograd.grad(ops.groupnorm_act(leaf, g, b, groups=8).sum(), leaf)[0]             # a broadcast gradient (stride 0)
    two = torch.autograd.grad(ops.groupnorm_act(leaf, g, b, groups=8), leaf, torch.ones_like(ref))[0]
    assert torch.equal(one, two)


def test_batch_invariance_and_repeat():
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(7, (24, 24), 320, torch.bfloat16, 9, dev)
    y, dx, dg, db = check_all(x, gamma, beta, dy, 32, True)
    y2, dx2, dg2, db2 = check_all(x, gamma, beta, dy, 32, True)
    assert all(torch.equal(a, b) for a, b in ((y, y2), (dx, dx2), (dg, dg2), (db, db2)))
    y3, dx3, _, _ = check_all(x[2:3], gamma, beta, dy[2:3], 32, True)
    assert torch.equal(y[2:3], y3) and torch.equal(dx[2:3], dx3)


def test_empty():
    dev = torch.device("cuda:0")
    gamma, beta = torch.ones(64, device=dev, requires_grad=True), torch.zeros(64, device=dev, requires_grad=True)
    for shape in ((0, 8, 64), (2, 0, 64)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        y = ops.groupnorm_act(x, gamma, beta, groups=8)
        gx, gg, gb = torch.autograd.grad(y, (x, gamma, beta), torch.zeros_like(y))
        assert y.shape == x.shape == gx.shape and not gg.any() and not gb.any()


def test_gradient_against_differences():
    """fp32, loss = sum(w * y): (loss(x + h e) - loss(x - h e)) / 2h in float64 of the reference formula against the kernel's gradient."""
    dev = torch.device("cuda:0")
    x, gamma, beta, w = data(1, (6,), 16, torch.float32, 21, dev)
    leaves = [t.detach().requires_grad_(True) for t in (x, gamma, beta)]
    got = torch.autograd.grad(ops.groupnorm_act(*leaves, groups=4), leaves, w)
    at = [t.detach().double().cpu() for t in (x, gamma, beta)]
    h = 1e-5
    for k, t in enumerate(at):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 5):
            keep = flat[i].item()
            vals = []
            for s in (h, -h):
                flat[i] = keep + s
                vals.append((reference(at[0].view(1, 6, 16), at[1], at[2], 4, 1e-5, True)[0] * w.double().cpu()).sum().item())
            flat[i] = keep
            diff = (vals[0] - vals[1]) / (2 * h)
            # second-order term h^2 * third derivative (a few units of |w| rstd^3) < 1e-8; fp32 arithmetic 1e-5 of the gradient's scale
            assert abs(diff - got[k].reshape(-1)[i].item()) <= 2e-5 * max(1.0, abs(diff)), (k, i)


def test_other_stream_and_graph():
    dev = torch.device("cuda:0")
    x, gamma, beta, dy = data(4, (16, 16), 320, torch.float16, 2, dev)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, gamma, beta)]
    y0 = ops.groupnorm_act(*leaves, groups=32)
    ref = [y0.detach().clone(), *(t.clone() for t in torch.autograd.grad(y0, leaves, dy))]
    del y0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.groupnorm_act(*leaves, groups=32)
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del y, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.groupnorm_act(*leaves, groups=32)
        out = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    for seed in (31, 32, 33):
        nx, ng, nb, nd = data(4, (16, 16), 320, torch.float16, seed, dev)
        with torch.no_grad():
            for t, n in zip((*leaves, dy), (nx, ng, nb, nd)):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        l2 = [t.detach().clone().requires_grad_(True) for t in leaves]
        y2 = ops.groupnorm_act(*l2, groups=32)
        assert all(torch.equal(a, b) for a, b in zip(out, [y2, *torch.autograd.grad(y2, l2, dy)]))
