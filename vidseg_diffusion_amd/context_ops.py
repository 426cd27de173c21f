"""Operators around the UNet's contexts that also carry gradients (csrc/norm_act.hip): reached as `ops.<name>`.

    groupnorm_act       GroupNorm (+ SiLU) of a channels-last map, any C / G, fp32 / fp16 / bf16; differentiable

Unlike the `*_a16` operators of ops.py, which run in the library's one 16-bit type, these take the type of their tensors.  They launch
asynchronously on torch's current stream of the tensors' device; scratch memory comes from torch's allocator call by call, so two streams
or two captured graphs never share any.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import VidsegError, call, ptr

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float

_lib.register({
    "vidseg_groupnorm_act_fwd": [_P, _L, _L, _I, _I, _L, _I, _I, _P, _P, _F, _I, _I, _P, _P, _P, _P, _L, _P],
    "vidseg_groupnorm_act_bwd": [_P, _L, _L, _P, _L, _L, _I, _I, _L, _I, _I, _P, _P, _P, _P, _I, _I, _P, _P, _P, _P, _L, _P],
})

F32 = torch.float32
_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _launch(device, name, *args):
    """call(name, *args, stream) on `device`, whichever device is the current one."""
    st = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        call(name, *args, st)
    else:
        with torch.cuda.device(device):
            call(name, *args, st)


def _need(cond, message):
    if not cond:
        raise VidsegError(message)


# ----------------------------------------------------------------------------- GroupNorm + activation
def norm_rows_per_chunk(HW, C):
    """Rows of one sample that a block reduces: about 40 K values (80 KB of fp16), at least 16 blocks a sample while there are rows for it.
    A function of HW and C alone, so a sample's statistics do not depend on the batch it is in."""
    return max(1, min(-(-40960 // C), -(-HW // 16)))


def _rows_of(x):
    """[B, ..., C] as rows: (tensor, B, HW, batch stride, row stride), copied only where the rows have no one stride."""
    B, C = x.shape[0], x.shape[-1]
    HW = 1
    for n in x.shape[1:-1]:
        HW *= n
    if C == 1 or x.stride(-1) == 1:
        dims = [(n, s) for n, s in zip(x.shape[1:-1], x.stride()[1:-1]) if n != 1]
        if all(dims[i][1] == dims[i + 1][0] * dims[i + 1][1] for i in range(len(dims) - 1)):
            row = dims[-1][1] if dims else C
            batch = x.stride(0) if B > 1 else HW * row
            if row >= C and batch >= 0:
                return x, B, HW, batch, row
    return x.contiguous(), B, HW, HW * C, C


def _groupnorm_act_fwd(x, gamma, beta, groups, eps, act, save):
    C = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x, B, HW, xb, xr = _rows_of(x)
    if y.numel() == 0:
        z = torch.zeros((2, B, groups), dtype=F32, device=x.device)
        return y, z[0], z[1]
    rows = norm_rows_per_chunk(HW, C)
    part = 2 * B * -(-HW // rows) * groups
    stats = torch.empty((2, B, groups), dtype=F32, device=x.device) if save else None
    scratch = torch.empty(part, dtype=F32, device=x.device)
    mean, rstd = (stats[0], stats[1]) if save else (None, None)
    _launch(x.device, "vidseg_groupnorm_act_fwd", x.data_ptr(), xb, xr, _DTYPE[x.dtype], B, HW, C, groups, gamma.data_ptr(), beta.data_ptr(), eps, act,
            rows, y.data_ptr(), ptr(mean), ptr(rstd), scratch.data_ptr(), part)
    return y, mean, rstd


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, groups, eps, act):
        y, mean, rstd = _groupnorm_act_fwd(x, gamma, beta, groups, eps, act, True)
        ctx.save_for_backward(x, gamma, beta, mean, rstd)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, gamma, beta, mean, rstd = ctx.saved_tensors
        C, G = x.shape[-1], ctx.groups
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if dx.numel() == 0:
            return dx, torch.zeros_like(gamma), torch.zeros_like(beta), None, None, None
        x, B, HW, xb, xr = _rows_of(x)
        dy, _, _, db, dr = _rows_of(dy)
        rows = norm_rows_per_chunk(HW, C)
        need = B * ((-(-HW // rows) + 1) * 2 * C + 2 * G)
        scratch = torch.empty(need, dtype=F32, device=x.device)
        dgb = torch.empty((2, C), dtype=F32, device=x.device)
        _launch(x.device, "vidseg_groupnorm_act_bwd", dy.data_ptr(), db, dr, x.data_ptr(), xb, xr, _DTYPE[x.dtype], B, HW, C, G, gamma.data_ptr(),
                beta.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ctx.act, rows, dx.data_ptr(), dgb[0].data_ptr(), dgb[1].data_ptr(),
                scratch.data_ptr(), need)
        return dx, dgb[0], dgb[1], None, None, None


def groupnorm_act(x, gamma, beta, *, groups=32, eps=1e-5, act=1):
    """act((x - mean_g) / sqrt(var_g + eps) * gamma + beta) over a channels-last map x [B, ..., C] (fp32 / fp16 / bf16; statistics and
    arithmetic in fp32, one rounding), group g = channels [g C / groups, (g + 1) C / groups) of one sample.  act: ops.ACT_SILU or
    ops.ACT_NONE.  gamma, beta: fp32 [C].  x may be a column slice of a wider map.  Differentiable in x, gamma and beta (once)
    (diffusionmodules/util.py:276-278 GroupNorm32, openaimodel.py:267-271)."""
    _need(x.dim() >= 2, "groupnorm_act: x must be [B, ..., C]")
    C = x.shape[-1]
    _need(x.dtype in _DTYPE, f"groupnorm_act: x of {x.dtype}: float32, float16 or bfloat16")
    _need(groups >= 1 and 1 <= C <= 8192 and C % groups == 0, f"groupnorm_act: {C} channels (at most 8192) in {groups} groups")
    _need(x.shape[0] <= 65535, f"groupnorm_act: {x.shape[0]} samples, at most 65535")
    _need(act in (0, 1), "groupnorm_act: act is ops.ACT_NONE or ops.ACT_SILU")
    _need(eps >= 0, "groupnorm_act: eps must not be negative")
    for n, t in (("gamma", gamma), ("beta", beta)):
        _need(t.dtype == F32 and t.dim() == 1 and t.shape[0] == C and t.stride(0) == 1 and t.device == x.device,
              f"groupnorm_act: {n} must be a contiguous fp32 [{C}] tensor on x's device")
    _need(x.is_cuda, "groupnorm_act: x must be a HIP device tensor (no CPU path)")
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad):
        return _GroupNormAct.apply(x, gamma, beta, groups, float(eps), act)
    return _groupnorm_act_fwd(x, gamma, beta, groups, float(eps), act, False)[0]
