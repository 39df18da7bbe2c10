"""Differential attention (csrc/diff_attn.h): the difference of two softmax maps over the same values,

    out = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v

per head, with a learned weight lam: what both maps spread over tokens that do not matter cancels.  It stands beside the aggregation net's ray attention
(network/ibrnet.py:160-204), which the render pass computes in its own kernel, for nets over more tokens than a ray has samples."""
import ctypes as C

import torch

from ._lib import PgrfDiffAttn, lib
from ._token import alike, dtype_code, on_device, on_gpu, ptr, require


def _aligned(t):
    """A tensor whose last axis is side by side and whose rows start at multiples of 16 bytes, with tokens and maps at most 2^22 values apart: t itself where it is one."""
    per = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % per == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])) and \
            all(t.stride(i) <= 1 << 22 for i in (1, 3) if i < t.dim() - 1 and t.shape[i] > 1):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t):
    return [0 if n == 1 else s for s, n in zip(t.stride(), t.shape)][:-1]


def _args(q, k, v, lam, mask, lengths, causal, scale):
    B, N, H, _, D = q.shape
    a = PgrfDiffAttn(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), ptr(mask), ptr(lengths))
    a.q_sb, a.q_sn, a.q_sh, a.q_sm = _strides(q)
    a.k_sb, a.k_sn, a.k_sh, a.k_sm = _strides(k)
    a.v_sb, a.v_sn, a.v_sh = _strides(v)
    if mask is not None:
        a.mask_sb = mask.stride(0) if B > 1 else 0
    a.dtype, a.lam_f32 = dtype_code(q, 'diff_attention'), int(lam.dtype == torch.float32)
    a.B, a.N, a.M, a.H, a.Hk, a.D, a.causal, a.scale = B, N, k.shape[1], H, k.shape[2], D, int(causal), scale
    return a


def _forward(q, k, v, lam, mask, lengths, causal, scale, train):
    B, N, H, _, D = q.shape
    M = k.shape[1]
    dev = q.device
    if B * N * M == 0:
        return torch.zeros(B, N, H, 2 * D, dtype=q.dtype, device=dev), None, None
    out = torch.empty(B, N, H, 2 * D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, H, 2, N, dtype=torch.float32, device=dev) if train else None
    maps = torch.empty(B, N, H, 2, 2 * D, dtype=torch.float32, device=dev) if train else None
    a = _args(q, k, v, lam, mask, lengths, causal, scale)
    a.out, a.lse, a.maps_out = out.data_ptr(), ptr(lse), ptr(maps)
    n = lib.pgrf_diff_attention_workspace_bytes(a.dtype, B, N, M, H, a.Hk, D)
    with on_device(dev) as stream:
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        a.workspace, a.workspace_bytes = ptr(ws), n
        lib.check(lib.pgrf_diff_attention(C.byref(a), stream))
    return out, lse, maps


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, mask, causal, scale):
        out, lse, maps = _forward(q, k, v, lam, mask, None, causal, scale, True)
        ctx.save_for_backward(q, k, v, lam, mask, lse, maps)
        ctx.call = (causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, mask, lse, maps = ctx.saved_tensors
        needs = ctx.needs_input_grad
        new = torch.zeros if lse is None else torch.empty
        make = lambda t, need: new(t.shape, dtype=t.dtype, device=t.device) if need else None
        both = needs[1] or needs[2]
        dq, dk, dv, dlam = make(q, needs[0]), make(k, both), make(v, both), make(lam, needs[3])
        if lse is not None:
            B, N, H, _, D = q.shape
            dout = _aligned(dout.contiguous())
            a = _args(q, k, v, lam, mask, None, *ctx.call)
            a.lse, a.maps_out = lse.data_ptr(), maps.data_ptr()
            n = lib.pgrf_diff_attention_backward_workspace_bytes(a.dtype, B, N, a.M, H, a.Hk, D)
            with on_device(q.device) as stream:
                ws = torch.empty(n, dtype=torch.uint8, device=q.device)
                a.workspace, a.workspace_bytes = ws.data_ptr(), n
                lib.check(lib.pgrf_diff_attention_backward(C.byref(a), dout.data_ptr(), ptr(dq), ptr(dk), ptr(dv), ptr(dlam), stream))
        return dq, dk if needs[1] else None, dv if needs[2] else None, dlam, None, None, None


def _check(who, q, k, v, lam, scale):
    for name, t, axes in (('q', q, '[B, N, H, 2, d]'), ('k', k, '[B, M, Hk, 2, d]'), ('v', v, '[B, M, Hk, 2 d]'), ('lam', lam, '[H]')):
        require(torch.is_tensor(t) and t.dim() == axes.count(',') + 1, who, f'{name} must be a tensor {axes}')
    dtype_code(q, who)
    alike(who, q.dtype, q.device, k=k, v=v)
    B, N, H, two, d = q.shape
    require(two == 2 and d in (32, 64, 128), who, f'q {tuple(q.shape)} must be [B, N, H, 2, d] with d 32, 64 or 128')
    Hk = k.shape[2]
    require(tuple(k.shape) == (B, k.shape[1], Hk, 2, d), who, f'k {tuple(k.shape)} must be [{B}, M, Hk, 2, {d}]')
    require(tuple(v.shape) == (B, k.shape[1], Hk, 2 * d), who, f'v {tuple(v.shape)} must be [{B}, {k.shape[1]}, {Hk}, {2 * d}]')
    require(H >= 1 and Hk >= 1 and H % Hk == 0, who, f'{H} query heads must be a multiple of {Hk} key heads')
    require(tuple(lam.shape) == (H,) and lam.device == q.device and lam.dtype in (q.dtype, torch.float32), who,
            f'lam must be [{H}] on {q.device}, float32 or of the type of q')
    scale = d ** -0.5 if scale is None else float(scale)
    require(0.0 < scale <= 1e30, who, 'scale must be positive')
    return scale


def diff_attention(q, k, v, lam, *, causal=False, key_mask=None, scale=None):
    """q [B, N, H, 2, d], k [B, M, Hk, 2, d], v [B, M, Hk, 2 d], lam [H] -> [B, N, H, 2 d].

    float32, bfloat16 or float16 (lam of that type or float32); d 32, 64 or 128; H a multiple of Hk: the query heads h Hk/H share a key head.  Any strides (rows
    that do not start at multiples of 16 bytes are copied first).  key_mask [B, M] bool, False: no query sees the key, and what it holds does not matter.
    causal: query i sees keys up to i + M - N, so the last query stands at the last key.  A query that sees no key gives 0.  scale: 1/sqrt(d) unless given.
    Softmax and sums are float; probabilities and score gradients are rounded to the tensors' type for the products behind them.  Gradients (first derivatives) to
    q, k, v and lam; they do not depend on scheduling."""
    who = 'diff_attention'
    scale = _check(who, q, k, v, lam, scale)
    if key_mask is not None:
        require(torch.is_tensor(key_mask) and key_mask.dtype == torch.bool and key_mask.device == q.device and tuple(key_mask.shape) == tuple(k.shape[:2]), who,
                f'key_mask must be a bool tensor {list(k.shape[:2])} on {q.device}')
    on_gpu(q, who)
    if key_mask is not None:
        key_mask = key_mask if key_mask.stride(-1) == 1 else key_mask.contiguous()
        key_mask = key_mask.view(torch.uint8)
    q, k, v, lam = _aligned(q), _aligned(k), _aligned(v), lam.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or lam.requires_grad):
        return _DiffAttention.apply(q, k, v, lam, key_mask, bool(causal), scale)
    return _forward(q, k, v, lam, key_mask, None, bool(causal), scale, False)[0]


def diff_attention_cached(q, k_cache, v_cache, lam, lengths, *, scale=None):
    """The same over a cache: k_cache [B, M, Hk, 2, d], v_cache [B, M, Hk, 2 d] of which the first lengths[b] keys count (lengths [B] int32 on the device,
    clamped to [0, M]; the rest may hold anything).  q [B, N, H, 2, d]: the last N tokens of each entry, causal among themselves: query i sees keys up to
    lengths[b] - N + i.  N = 1 is the step of a served model.  The lengths are read on the device, so a captured step follows them.  No gradients."""
    who = 'diff_attention_cached'
    scale = _check(who, q, k_cache, v_cache, lam, scale)
    require(torch.is_tensor(lengths) and lengths.dtype == torch.int32 and lengths.device == q.device and tuple(lengths.shape) == (q.shape[0],), who,
            f'lengths must be an int32 tensor [{q.shape[0]}] on {q.device}')
    require(not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_cache, v_cache, lam))), who,
            'no gradients over a cache: call it under torch.no_grad(), or diff_attention with a key_mask')
    on_gpu(q, who)
    return _forward(_aligned(q), _aligned(k_cache), _aligned(v_cache), lam.contiguous(), None, lengths.contiguous(), True, scale, False)[0]
