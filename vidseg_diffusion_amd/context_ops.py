"""Operators around the UNet's contexts (csrc/norm_act.hip, csrc/context_attn.hip): reached as `ops.<name>`.

    groupnorm_act       GroupNorm (+ SiLU) of a channels-last map, any C / G, fp32 / fp16 / bf16; differentiable
    cross_attention     attention to an encoder's states of another length, per-sample lengths / key mask, heads of 8..128, grouped heads;
                        differentiable
    prefix_attention    attention of a batch to keys that all samples share and to each sample's own keys

Unlike the `*_a16` operators of ops.py, which run in the library's one 16-bit type, these take the type of their tensors.  They launch
asynchronously on torch's current stream of the tensors' device; scratch memory comes from torch's allocator call by call, so two streams
or two captured graphs never share any.  A backward pass can be captured too, on leaves of which no eager graph is alive: torch ties a leaf's
gradient to the stream on which the leaf was first used, and a captured pass cannot wait for another stream.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import VidsegError, call, ptr

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float

_lib.register({
    "vidseg_groupnorm_act_fwd": [_P, _L, _L, _I, _I, _L, _I, _I, _P, _P, _F, _I, _I, _P, _P, _P, _P, _L, _P],
    "vidseg_context_attention_scratch_kib": [_I, _I, _I, _I, _I, _I, _I],
    "vidseg_context_attention_fwd": [_P, _L, _L, _L] + [_P, _L, _L] * 2 + [_P, _L, _L, _L] * 2 + [_P, _P, _L, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _I, _P, _L, _P],
    "vidseg_context_attention_bwd_scratch_kib": [_I, _I, _I, _I, _I, _I, _I],
    "vidseg_context_attention_bwd": [_P, _L, _L, _L] * 4 + [_P, _P, _L, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _F, _P, _L, _P],
    "vidseg_groupnorm_act_bwd": [_P, _L, _L, _P, _L, _L, _I, _I, _L, _I, _I, _P, _P, _P, _P, _I, _I, _P, _P, _P, _P, _L, _P],
})

F32 = torch.float32
_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_raw_stream = torch._C._cuda_getCurrentRawStream              # the handle of torch.cuda.current_stream(device) without the Python object around it


def _launch(device, name, *args):
    """call(name, *args, stream) on `device`, whichever device is the current one."""
    if device.index == torch.cuda.current_device():
        call(name, *args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            call(name, *args, _raw_stream(device.index))


def _need(cond, message, *args):
    if not cond:
        raise VidsegError(message % args if args else message)


def _no_tangents(name, *tensors):
    """Refuses dual tensors: they ask for no gradient, and a result without a tangent would read as a derivative of zero."""
    if forward_ad._current_level >= 0:
        _need(all(forward_ad.unpack_dual(t).tangent is None for t in tensors), "%s: carries no forward-mode derivatives", name)


# ----------------------------------------------------------------------------- GroupNorm + activation
def norm_rows_per_chunk(HW, C):
    """Rows of one sample that a block reduces: about 40 K values (80 KB of fp16), at least 16 blocks a sample while there are rows for it.
    A function of HW and C alone, so a sample's statistics do not depend on the batch it is in."""
    return max(1, min(-(-40960 // C), -(-HW // 16)))


def _rows_of(x):
    """[B, ..., C] as rows: (tensor, B, HW, batch stride, row stride), copied only where the rows have no one stride."""
    shape = x.shape
    B, C = shape[0], shape[-1]
    HW = 1
    for n in shape[1:-1]:
        HW *= n
    if x.is_contiguous():
        return x, B, HW, HW * C, C
    if C == 1 or x.stride(-1) == 1:
        dims = [(n, s) for n, s in zip(shape[1:-1], x.stride()[1:-1]) if n != 1]
        if all(dims[i][1] == dims[i + 1][0] * dims[i + 1][1] for i in range(len(dims) - 1)):
            row = dims[-1][1] if dims else C
            batch = x.stride(0) if B > 1 else HW * row
            if row >= C and batch >= 0:
                return x, B, HW, batch, row
    return x.contiguous(), B, HW, HW * C, C


def _groupnorm_act_fwd(x, gamma, beta, groups, eps, act, save):
    device = x.device
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    x, B, HW, xb, xr = _rows_of(x)
    C = x.shape[-1]
    if B * HW == 0:
        return y, torch.zeros(2 * B * groups, dtype=F32, device=device)
    rows = norm_rows_per_chunk(HW, C)
    part = 2 * B * -(-HW // rows) * groups
    stats = torch.empty(2 * B * groups + part, dtype=F32, device=device)        # means, 1 / standard deviations, scratch behind them
    mean = stats.data_ptr()
    rstd = mean + 4 * B * groups
    _launch(device, "vidseg_groupnorm_act_fwd", x.data_ptr(), xb, xr, _DTYPE[x.dtype], B, HW, C, groups, gamma.data_ptr(), beta.data_ptr(), eps, act,
            rows, y.data_ptr(), mean if save else None, rstd if save else None, rstd + 4 * B * groups, part)
    return y, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, groups, eps, act):
        y, stats = _groupnorm_act_fwd(x, gamma, beta, groups, eps, act, True)
        ctx.save_for_backward(x, gamma, beta, stats)
        ctx.how = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, gamma, beta, stats = ctx.saved_tensors
        G, act = ctx.how
        device = x.device
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        x, B, HW, xb, xr = _rows_of(x)
        dy, _, _, db, dr = _rows_of(dy)
        C = x.shape[-1]
        if B * HW == 0:
            return dx, torch.zeros_like(gamma), torch.zeros_like(beta), None, None, None
        rows = norm_rows_per_chunk(HW, C)
        need = 2 * B * -(-HW // rows) * (C + G)
        scratch = torch.empty(need, dtype=F32, device=device)
        dgamma = torch.empty(C, dtype=F32, device=device)
        dbeta = torch.empty(C, dtype=F32, device=device)
        at = stats.data_ptr()
        _launch(device, "vidseg_groupnorm_act_bwd", dy.data_ptr(), db, dr, x.data_ptr(), xb, xr, _DTYPE[x.dtype], B, HW, C, G, gamma.data_ptr(),
                beta.data_ptr(), at, at + 4 * B * G, act, rows, dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), scratch.data_ptr(), need)
        return dx, dgamma, dbeta, None, None, None


def groupnorm_act(x, gamma, beta, *, groups=32, eps=1e-5, act=1):
    """act((x - mean_g) / sqrt(var_g + eps) * gamma + beta) over a channels-last map x [B, ..., C] (fp32 / fp16 / bf16; statistics and
    arithmetic in fp32, one rounding), group g = channels [g C / groups, (g + 1) C / groups) of one sample.  act: ops.ACT_SILU or
    ops.ACT_NONE.  gamma, beta: fp32 [C].  x may be a column slice of a wider map.  Differentiable in x, gamma and beta (once, in
    reverse mode) (diffusionmodules/util.py:276-278 GroupNorm32, openaimodel.py:267-271)."""
    shape = x.shape
    _need(len(shape) >= 2, "groupnorm_act: x must be [B, ..., C]")
    C = shape[-1]
    _need(x.dtype in _DTYPE, "groupnorm_act: x of %s: float32, float16 or bfloat16", x.dtype)
    _need(groups >= 1 and 1 <= C <= 8192 and C % groups == 0, "groupnorm_act: %d channels (at most 8192) in %d groups", C, groups)
    _need(shape[0] <= 65535, "groupnorm_act: %d samples, at most 65535", shape[0])
    _need(act == 0 or act == 1, "groupnorm_act: act is ops.ACT_NONE or ops.ACT_SILU")
    _need(eps >= 0, "groupnorm_act: eps must not be negative")
    for n, t in (("gamma", gamma), ("beta", beta)):
        _need(t.dtype == F32 and t.shape == (C,) and t.stride(0) == 1 and t.device == x.device,
              "groupnorm_act: %s must be a contiguous fp32 [%d] tensor on x's device", n, C)
    _no_tangents("groupnorm_act", x, gamma, beta)
    _need(x.is_cuda, "groupnorm_act: x must be a HIP device tensor (no CPU path)")
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad):
        return _GroupNormAct.apply(x, gamma, beta, groups, float(eps), act)
    return _groupnorm_act_fwd(x, gamma, beta, groups, float(eps), act, False)[0]


# ----------------------------------------------------------------------------- attention to contexts
def _heads_of(t, d):
    """[.., N, heads * d] or [.., N, heads, d] as (tensor, pointer, first, row and head stride): a copy only where the last dimension is not contiguous,
    16-byte pieces are not aligned or rows lie 2^24 elements and more apart."""
    for copied in (False, True):
        st = t.stride()
        n, h = (st[-2], d) if len(st) == 3 else (st[-3], st[-2])
        at = t.data_ptr()
        if st[-1] == 1 and not (st[0] | n | h) & 7 and not at & 15 and n < 1 << 24:
            return t, at, st[0] if t.shape[0] > 1 else 0, n, h
        _need(not copied, "rows of %d elements cannot be laid out for the kernels", n)
        t = t.clone(memory_format=torch.contiguous_format)


def _attention_shapes(name, q, heads, kv_heads, kv):
    """Checks q [B, Nq, heads * d] (or [B, Nq, heads, d]) and the tensors kv = (name, tensor, leading dimensions); returns d, kv_heads."""
    shape = q.shape
    _need(len(shape) == 3 or len(shape) == 4, "%s: q must be [B, Nq, heads * d] or [B, Nq, heads, d]", name)
    _need(q.dtype == torch.float16 or q.dtype == torch.bfloat16, "%s: q of %s: float16 or bfloat16", name, q.dtype)
    four = len(shape) == 4
    _need(heads >= 1 and (shape[2] == heads if four else shape[2] % heads == 0), "%s: q of shape %s does not hold %d heads", name, tuple(shape), heads)
    d = shape[3] if four else shape[2] // heads
    kv_heads = heads if kv_heads is None else kv_heads
    _need(heads <= 1024, "%s: %d heads, at most 1024", name, heads)
    _need(kv_heads >= 1 and heads % kv_heads == 0, "%s: %d heads on %d key heads", name, heads, kv_heads)
    _need(8 <= d <= 128 and d % 8 == 0, "%s: head width %d: a multiple of 8 up to 128", name, d)
    for n, t, lead in kv:
        s = t.shape
        _need(t.dtype == q.dtype, "%s: %s of %s, q of %s", name, n, t.dtype, q.dtype)
        _need(t.device == q.device, "%s: %s on %s, q on %s", name, n, t.device, q.device)
        _need(s[1 + lead:] == (kv_heads, d) if len(s) == 3 + lead else len(s) == 2 + lead and s[-1] == kv_heads * d,
              "%s: %s of shape %s does not hold rows of %d heads of %d", name, n, tuple(s), kv_heads, d)
    return d, kv_heads


def _lengths(name, t, B, device):
    _need(t.dtype == torch.int32 and t.shape == (B,) and t.is_contiguous() and t.device == device,
          "%s: k_lens must be a contiguous int32 [%d] tensor on q's device", name, B)


def _mask(key_mask):
    """Pointer and sample stride of a key mask."""
    if key_mask is None:
        return None, 0
    return key_mask.data_ptr(), key_mask.stride(0) if key_mask.shape[0] > 1 else 0


def _context_attention(q, k_prefix, v_prefix, k, v, heads, kv_heads, d, k_lens, key_mask, scale, causal, want_lse, out_lo=None):
    B, Nq = q.shape[:2]
    device = q.device
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((B, heads, Nq), dtype=F32, device=device) if want_lse else None
    if B * Nq == 0:
        return out, lse
    q, qp, qb, qn, qh = _heads_of(q, d)
    Np, Nk = 0, k.shape[1]
    pre, own = (None, 0, 0) * 2, (None, 0, 0, 0) * 2
    if k_prefix is not None and k_prefix.shape[0]:
        Np = k_prefix.shape[0]
        kp, a, _, b, c = _heads_of(k_prefix[None], d)
        vp, e, _, f, g = _heads_of(v_prefix[None], d)
        pre = (a, b, c, e, f, g)
    if Nk:
        k, *ks = _heads_of(k, d)
        v, *vs = _heads_of(v, d)
        own = (*ks, *vs)
    kib = _lib.lib().vidseg_context_attention_scratch_kib(B, Nq, Np, Nk, heads, kv_heads, d)
    scratch = torch.empty(kib * 256, dtype=F32, device=device) if kib > 0 else None
    _launch(device, "vidseg_context_attention_fwd", qp, qb, qn, qh, *pre, *own, ptr(k_lens), *_mask(key_mask), out.data_ptr(), ptr(out_lo), ptr(lse),
            _DTYPE[q.dtype], B, Nq, Np, Nk, heads, kv_heads, d, scale, causal, ptr(scratch), max(kib, 0))
    return out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, heads, kv_heads, d, k_lens, key_mask, scale):
        # over 128 keys the backward pass takes sum(do * o) from the saved result, to more bits than its type has; below, it has no use for it
        left = torch.empty_like(q, memory_format=torch.contiguous_format) if k.shape[1] > 128 else None
        out, lse = _context_attention(q, None, None, k, v, heads, kv_heads, d, k_lens, key_mask, scale, 0, True, left)
        ctx.save_for_backward(q, k, v, k_lens, key_mask, None if left is None else out, left, lse)
        ctx.how = heads, kv_heads, d, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 9
        q, k, v, k_lens, key_mask, out, left, lse = ctx.saved_tensors
        heads, kv_heads, d, scale = ctx.how
        device, dtype = q.device, q.dtype
        (B, Nq), (Bk, Nk) = q.shape[:2], k.shape[:2]
        if B * Nq * Nk == 0:
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), *(None,) * 6)
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        dk = dv = None
        if Nk <= 128 or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dk = torch.empty_like(k, memory_format=torch.contiguous_format)
            dv = torch.empty_like(v, memory_format=torch.contiguous_format)
        dout, *gs = _heads_of(dout, d)
        q, *qs = _heads_of(q, d)
        k, *ks = _heads_of(k, d)
        v, *vs = _heads_of(v, d)
        kib = _lib.lib().vidseg_context_attention_bwd_scratch_kib(B, Bk, Nq, Nk, heads, kv_heads, d)
        scratch = torch.empty(kib * 256, dtype=F32, device=device) if kib > 0 else None
        _launch(device, "vidseg_context_attention_bwd", *gs, *qs, *ks, *vs, ptr(k_lens), *_mask(key_mask), ptr(out), ptr(left), lse.data_ptr(), dq.data_ptr(),
                ptr(dk), ptr(dv), _DTYPE[dtype], B, Bk, Nq, Nk, heads, kv_heads, d, scale, ptr(scratch), max(kib, 0))
        return dq, dk, dv, None, None, None, None, None, None


def cross_attention(q, k, v, heads, *, kv_heads=None, k_lens=None, key_mask=None, scale=None, return_lse=False):
    """softmax(scale q k^T over the keys that exist) v, heads side by side: q [B, Nq, heads * d], k / v [B or 1, Nk, kv_heads * d] (the heads may also
    be a dimension of their own, in any order of strides; d a multiple of 8 up to 128, at most 1024 heads; fp16 / bf16; scale defaults to d^-1/2).
    Scores, maxima, sums and accumulators are fp32; probabilities and, in the gradients, dp - D times them are rounded once to the tensors' type before the
    product that takes them, so a result is off by up to about two half steps of that type where attention in fp32 would be off by one.
    Query head h reads key head h * kv_heads // heads.  One sample of k / v serves the whole batch.  A key exists if it lies below k_lens[b] (int32 [B] on the device)
    and key_mask[b or 0, key] (bool) is true; what k / v hold elsewhere, NaN included, reaches nothing, and a query without any key gets zeros.
    return_lse: also log(sum exp) of the scores, fp32 [B, heads, Nq] (-inf without a key).  Differentiable (once, in reverse mode) in q, k and v,
    not through the log-sum-exp.  Gradients of one shared k / v are summed over the batch  (attention.py:286-364)."""
    name = "cross_attention"
    d, kv_heads = _attention_shapes(name, q, heads, kv_heads, (("k", k, 1), ("v", v, 1)))
    B, sk = q.shape[0], k.shape
    _need(sk[0] == B or sk[0] == 1, "%s: k and v hold %d samples, q %d", name, sk[0], B)
    _need(sk[:2] == v.shape[:2], "%s: k of shape %s, v of shape %s", name, tuple(sk), tuple(v.shape))
    if k_lens is not None:
        _lengths(name, k_lens, B, q.device)
    if key_mask is not None:
        _need(key_mask.dtype == torch.bool and key_mask.dim() == 2 and key_mask.shape[0] in (1, B) and key_mask.shape[1] == sk[1] and key_mask.device == q.device
              and (key_mask.stride(1) == 1 or sk[1] == 1), "%s: key_mask must be a bool [%d or 1, %d] tensor with contiguous rows on q's device", name, B, sk[1])
    scale = d ** -0.5 if scale is None else float(scale)
    _need(0 < scale < float("inf"), "%s: scale must be positive and finite", name)
    _no_tangents(name, q, k, v)
    _need(q.is_cuda, "%s: q must be a HIP device tensor (no CPU path)", name)
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
    causal: the queries are the last Nq of the k_lens[b] own tokens, and query i sees own keys up to its own position k_lens[b] - Nq + i.  Later keys
    of the k_lens[b] have probability zero for it, but their values have to be finite: zero times NaN or infinity is NaN.
    No gradients: the call is refused where one is asked for."""
    name = "prefix_attention"
    d, kv_heads = _attention_shapes(name, q, heads, kv_heads, (("k", k, 1), ("v", v, 1), ("k_prefix", k_prefix, 0), ("v_prefix", v_prefix, 0)))
    B, sk = q.shape[0], k.shape
    _need(sk[0] == B, "%s: k and v hold %d samples, q %d", name, sk[0], B)
    _need(sk[:2] == v.shape[:2], "%s: k of shape %s, v of shape %s", name, tuple(sk), tuple(v.shape))
    _need(k_prefix.shape[0] == v_prefix.shape[0], "%s: prefix of %d keys and %d values", name, k_prefix.shape[0], v_prefix.shape[0])
    if k_lens is not None:
        _lengths(name, k_lens, B, q.device)
    scale = d ** -0.5 if scale is None else float(scale)
    _need(0 < scale < float("inf"), "%s: scale must be positive and finite", name)
    _need(not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_prefix, v_prefix, k, v))),
          "%s: carries no gradients (use it under torch.no_grad())", name)
    _no_tangents(name, q, k_prefix, v_prefix, k, v)
    _need(q.is_cuda, "%s: q must be a HIP device tensor (no CPU path)", name)
    out, lse = _context_attention(q, k_prefix, v_prefix, k, v, heads, kv_heads, d, k_lens, None, scale, int(causal), return_lse)
    return (out, lse) if return_lse else out
