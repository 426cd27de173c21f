"""Operators around the UNet's contexts (csrc/norm_act.hip, csrc/context_attn.hip): reached as `ops.<name>`.

    groupnorm_act       GroupNorm (+ SiLU) of a channels-last map, any C / G, fp32 / fp16 / bf16; differentiable
    cross_attention     attention to an encoder's states of another length, per-sample lengths / key mask, heads of 8..128, grouped heads;
                        differentiable
    prefix_attention    attention of a batch to keys that all samples share and to each sample's own keys

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
    "vidseg_context_attention_scratch_kib": [_I, _I, _I, _I, _I, _I, _I],
    "vidseg_context_attention_fwd": [_P, _L, _L, _L] + [_P, _L, _L] * 2 + [_P, _L, _L, _L] * 2 + [_P, _P, _L, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _I, _P, _L, _P],
    "vidseg_context_attention_bwd_scratch_kib": [_I, _I, _I, _I, _I, _I, _I],
    "vidseg_context_attention_bwd": [_P, _L, _L, _L] * 4 + [_P, _P, _L, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _P, _L, _P],
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


# ----------------------------------------------------------------------------- attention to contexts
def _heads_of(name, t, heads, d):
    """[B, N, heads * d] or [B, N, heads, d] as (tensor, batch, row, head strides); copied only where the last dimension is not contiguous or 16-byte
    pieces are not aligned."""
    if t.dim() == 3:
        t = t.unflatten(2, (heads, d))
    st = t.stride()
    if (st[3] != 1 and d > 1) or st[0] % 8 or st[1] % 8 or st[2] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st = t.stride()
    return t, st[0] if t.shape[0] > 1 else 0, st[1], st[2]


def _attention_shapes(name, q, heads, kv_heads, kv):
    """Checks q [B, Nq, heads * d] (or [B, Nq, heads, d]) and the tensors kv = {name: (tensor, batch sizes allowed or None)}; returns d, kv_heads."""
    _need(q.dim() in (3, 4), f"{name}: q must be [B, Nq, heads * d] or [B, Nq, heads, d]")
    _need(q.dtype in (torch.float16, torch.bfloat16), f"{name}: q of {q.dtype}: float16 or bfloat16")
    _need(heads >= 1 and (q.shape[2] == heads if q.dim() == 4 else q.shape[2] % heads == 0), f"{name}: q of shape {tuple(q.shape)} does not hold {heads} heads")
    d = q.shape[3] if q.dim() == 4 else q.shape[2] // heads
    kv_heads = heads if kv_heads is None else kv_heads
    _need(kv_heads >= 1 and heads % kv_heads == 0, f"{name}: {heads} heads on {kv_heads} key heads")
    _need(8 <= d <= 128 and d % 8 == 0, f"{name}: head width {d}: a multiple of 8 up to 128")
    for n, (t, batches) in kv.items():
        lead = 1 if batches else 0
        _need(t.dtype == q.dtype, f"{name}: {n} of {t.dtype}, q of {q.dtype}")
        _need(t.device == q.device, f"{name}: {n} on {t.device}, q on {q.device}")
        _need(t.dim() in (2 + lead, 3 + lead) and (tuple(t.shape[1 + lead:]) == (kv_heads, d) if t.dim() == 3 + lead else t.shape[-1] == kv_heads * d),
              f"{name}: {n} of shape {tuple(t.shape)} does not hold rows of {kv_heads} heads of {d}")
        _need(not batches or t.shape[0] in batches, f"{name}: {n} holds {t.shape[0]} samples, q {q.shape[0]}")
    return d, kv_heads


def _lengths(name, t, B, device):
    _need(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == B and t.is_contiguous() and t.device == device,
          f"{name}: k_lens must be a contiguous int32 [{B}] tensor on q's device")


def _context_attention(q, k_prefix, v_prefix, k, v, heads, kv_heads, d, k_lens, key_mask, scale, causal, want_lse):
    B, Nq = q.shape[:2]
    out = torch.empty((B, Nq, heads, d) if q.dim() == 4 else (B, Nq, heads * d), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, heads, Nq), dtype=F32, device=q.device) if want_lse else None
    if out.numel() == 0:
        return out, lse
    q, qb, qn, qh = _heads_of("q", q, heads, d)
    Np = Nk = 0
    pre, own = (None, 0, 0) * 2, (None, 0, 0, 0) * 2
    if k_prefix is not None and k_prefix.shape[0]:
        Np = k_prefix.shape[0]
        kp, _, a, b = _heads_of("k_prefix", k_prefix[None], kv_heads, d)
        vp, _, e, f = _heads_of("v_prefix", v_prefix[None], kv_heads, d)
        pre = (kp.data_ptr(), a, b, vp.data_ptr(), e, f)
    if k.shape[1]:
        Nk = k.shape[1]
        k, kb, kn, kh = _heads_of("k", k, kv_heads, d)
        v, vb, vn, vh = _heads_of("v", v, kv_heads, d)
        own = (k.data_ptr(), kb, kn, kh, v.data_ptr(), vb, vn, vh)
    kib = _lib.lib().vidseg_context_attention_scratch_kib(B, Nq, Np, Nk, heads, kv_heads, d)
    scratch = torch.empty(kib * 256, dtype=F32, device=q.device) if kib > 0 else None
    mb = key_mask.stride(0) if key_mask is not None and key_mask.shape[0] > 1 else 0
    _launch(q.device, "vidseg_context_attention_fwd", q.data_ptr(), qb, qn, qh, *pre, *own, ptr(k_lens), ptr(key_mask), mb, out.data_ptr(), ptr(lse),
            _DTYPE[q.dtype], B, Nq, Np, Nk, heads, kv_heads, d, scale, causal, ptr(scratch), max(kib, 0))
    return out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, heads, kv_heads, d, k_lens, key_mask, scale):
        out, lse = _context_attention(q, None, None, k, v, heads, kv_heads, d, k_lens, key_mask, scale, 0, True)
        ctx.save_for_backward(q, k, v, k_lens, key_mask, out, lse)
        ctx.sizes = heads, kv_heads, d, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        none = (None,) * 6
        if dout is None:
            return (None, None, None, *none)
        q, k, v, k_lens, key_mask, out, lse = ctx.saved_tensors
        heads, kv_heads, d, scale = ctx.sizes
        (B, Nq), (Bk, Nk) = q.shape[:2], k.shape[:2]
        if out.numel() == 0 or Nk == 0:
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), *none)
        want_kv = Nk <= 128 or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if on else None for t, on in ((q, True), (k, want_kv), (v, want_kv)))
        operands = ()
        for n, t, h in (("dout", dout, heads), ("q", q, heads), ("k", k, kv_heads), ("v", v, kv_heads)):
            t, *strides = _heads_of(n, t, h, d)
            operands += ((t, *strides),)
        flat = [x for t, *strides in operands for x in (t.data_ptr(), *strides)]
        kib = _lib.lib().vidseg_context_attention_bwd_scratch_kib(B, Bk, Nq, Nk, heads, kv_heads, d)
        scratch = torch.empty(kib * 256, dtype=F32, device=q.device) if kib > 0 else None
        mb = key_mask.stride(0) if key_mask is not None and key_mask.shape[0] > 1 else 0
        _launch(q.device, "vidseg_context_attention_bwd", *flat, ptr(k_lens), ptr(key_mask), mb, out.data_ptr(), lse.data_ptr(), dq.data_ptr(), ptr(dk), ptr(dv),
                _DTYPE[q.dtype], B, Bk, Nq, Nk, heads, kv_heads, d, scale, ptr(scratch), max(kib, 0))
        return (dq, dk, dv, *none)


def cross_attention(q, k, v, heads, *, kv_heads=None, k_lens=None, key_mask=None, scale=None, return_lse=False):
    """softmax(scale q k^T over the keys that exist) v, heads side by side: q [B, Nq, heads * d], k / v [B or 1, Nk, kv_heads * d] (the heads may also
    be a dimension of their own, in any order of strides; d a multiple of 8 up to 128; fp16 / bf16, fp32 inside; scale defaults to d^-1/2).
    Query head h reads key head h * kv_heads // heads.  One sample of k / v serves the whole batch.  A key exists if it lies below k_lens[b] (int32 [B] on the device)
    and key_mask[b or 0, key] (bool) is true; what k / v hold elsewhere, NaN included, reaches nothing, and a query without any key gets zeros.
    return_lse: also log(sum exp) of the scores, fp32 [B, heads, Nq] (-inf without a key).  Differentiable (once) in q, k and v, not through the
    log-sum-exp; in fp16 the gradients hold for |v| below 500.  Gradients of one shared k / v are summed over the batch  (attention.py:286-364)."""
    name = "cross_attention"
    B = q.shape[0] if q.dim() else 0
    d, kv_heads = _attention_shapes(name, q, heads, kv_heads, {"k": (k, (1, B)), "v": (v, (1, B))})
    _need(k.shape[:2] == v.shape[:2], f"{name}: k of shape {tuple(k.shape)}, v of shape {tuple(v.shape)}")
    if k_lens is not None:
        _lengths(name, k_lens, B, q.device)
    if key_mask is not None:
        _need(key_mask.dtype == torch.bool and key_mask.dim() == 2 and key_mask.shape[0] in (1, B) and key_mask.shape[1] == k.shape[1] and key_mask.device == q.device
              and (key_mask.stride(1) == 1 or key_mask.shape[1] == 1), f"{name}: key_mask must be a bool [{B} or 1, {k.shape[1]}] tensor with contiguous rows on q's device")
    scale = d ** -0.5 if scale is None else float(scale)
    _need(0 < scale < float("inf"), f"{name}: scale must be positive and finite")
    _need(q.is_cuda, f"{name}: q must be a HIP device tensor (no CPU path)")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _CrossAttention.apply(q, k, v, heads, kv_heads, d, k_lens, key_mask, scale)
    else:
        out, lse = _context_attention(q, None, None, k, v, heads, kv_heads, d, k_lens, key_mask, scale, 0, return_lse)
    return (out, lse) if return_lse else out


def prefix_attention(q, k_prefix, v_prefix, k, v, heads, *, kv_heads=None, k_lens=None, causal=False, scale=None, return_lse=False):
    """Attention of a batch to Np keys that all its samples share and to each sample's own keys, as one softmax over both: q [B, Nq, heads * d],
    k_prefix / v_prefix [Np, kv_heads * d], k / v [B, Nk, kv_heads * d] with k_lens[b] keys in use (all without k_lens); layouts and types as in
    cross_attention, Np and Nk may be 0.  The prefix is read once for all samples where they bring few queries each (single tokens behind one
    prompt), and through each XCD's cache where they bring many (frames over an anchor frame's keys).
    causal: the queries are the last Nq of the k_lens[b] own tokens, and query i sees own keys up to its own position k_lens[b] - Nq + i.
    No gradients: the call is refused where one is asked for."""
    name = "prefix_attention"
    B = q.shape[0] if q.dim() else 0
    d, kv_heads = _attention_shapes(name, q, heads, kv_heads, {"k": (k, (B,)), "v": (v, (B,)), "k_prefix": (k_prefix, None), "v_prefix": (v_prefix, None)})
    _need(k.shape[:2] == v.shape[:2], f"{name}: k of shape {tuple(k.shape)}, v of shape {tuple(v.shape)}")
    _need(k_prefix.shape[0] == v_prefix.shape[0], f"{name}: prefix of {k_prefix.shape[0]} keys and {v_prefix.shape[0]} values")
    if k_lens is not None:
        _lengths(name, k_lens, B, q.device)
    scale = d ** -0.5 if scale is None else float(scale)
    _need(0 < scale < float("inf"), f"{name}: scale must be positive and finite")
    _need(not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_prefix, v_prefix, k, v))), f"{name}: carries no gradients (use it under torch.no_grad())")
    _need(q.is_cuda, f"{name}: q must be a HIP device tensor (no CPU path)")
    out, lse = _context_attention(q, k_prefix, v_prefix, k, v, heads, kv_heads, d, k_lens, None, scale, int(causal), return_lse)
    return (out, lse) if return_lse else out
