"""Differential attention (csrc/diff_attn.h): the difference of two softmax maps over the same values,

    out = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v

per head, with a learned weight lam: what both maps spread over tokens that do not matter cancels.  It stands beside the aggregation net's ray attention
(network/ibrnet.py:160-204), which the render pass computes in its own kernel, for nets over more tokens than a ray has samples."""
from functools import lru_cache

import torch

from ._token import DIFF_ATTN, DTYPES, alike, entry, first_derivatives_only, launch, no_tangents, on_gpu, ptr, refuse, require


def _aligned(t):
    """A tensor whose last axis is side by side and whose rows start at multiples of 16 bytes, with tokens and maps at most 2^22 values apart: t itself where it is one."""
    s = t.stride()
    odd = 0
    for x in s[:-1]:
        odd |= x
    if s[-1] == 1 and odd % (16 // t.element_size()) == 0 and s[1] <= 1 << 22 and (len(s) < 5 or s[3] <= 1 << 22) and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()                              # (a contiguous tensor's rows are multiples of 16 bytes; axes of one may have any stride)
    s = t.stride()
    if t.data_ptr() % 16 or (t.shape[1] > 1 and s[1] > 1 << 22) or any(x % (16 // t.element_size()) for x in s[:-1]):
        t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    return t


@lru_cache(maxsize=256)
def _of_sizes(name, *sizes):
    return entry(name)(*sizes)


def _pack(q, k, v, lam, mask, lengths, causal, scale, out, lse, maps, ws, ws_bytes):
    B, N, H, _, D = q.shape
    q0, q1, q2, q3, _ = q.stride()
    k0, k1, k2, k3, _ = k.stride()
    v0, v1, v2, _ = v.stride()
    return DIFF_ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), 0 if mask is None else mask.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                          0 if out is None else out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if maps is None else maps.data_ptr(), 0 if ws is None else ws.data_ptr(),
                          ws_bytes, q0, q1, q2, q3, k0, k1, k2, k3, v0, v1, v2, 0 if mask is None or B == 1 else mask.stride(0),
                          DTYPES[q.dtype], lam.dtype == torch.float32, B, N, k.shape[1], H, k.shape[2], D, causal, scale)


def _forward(q, k, v, lam, mask, lengths, causal, scale, train):
    B, N, H, _, D = q.shape
    M = k.shape[1]
    dev = q.device
    if B * N * M == 0:
        return torch.zeros(B, N, H, 2 * D, dtype=q.dtype, device=dev), None, None
    out = torch.empty(B, N, H, 2 * D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, H, 2, N, dtype=torch.float32, device=dev) if train else None
    maps = torch.empty(B, N, H, 2, 2 * D, dtype=torch.float32, device=dev) if train and _of_sizes('pgrf_diff_attention_keeps_maps', DTYPES[q.dtype], M) else None
    n = _of_sizes('pgrf_diff_attention_workspace_bytes', DTYPES[q.dtype], B, N, M, H, k.shape[2], D)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    launch(dev, 'pgrf_diff_attention', _pack(q, k, v, lam, mask, lengths, causal, scale, out, lse, maps, ws, n))
    return out, lse, maps


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, mask, causal, scale):
        out, lse, maps = _forward(q, k, v, lam, mask, None, causal, scale, True)
        ctx.save_for_backward(q, k, v, lam, mask, lse, maps)
        ctx.call = (causal, scale)
        return out

    @staticmethod
    @first_derivatives_only
    def backward(ctx, dout):
        q, k, v, lam, mask, lse, maps = ctx.saved_tensors
        needs = ctx.needs_input_grad
        new = torch.zeros if lse is None else torch.empty
        make = lambda t, need: new(t.shape, dtype=t.dtype, device=t.device) if need else None
        both = needs[1] or needs[2]
        dq, dk, dv, dlam = make(q, needs[0]), make(k, both), make(v, both), make(lam, needs[3])
        if lse is not None:
            B, N, H, _, D = q.shape
            dout = dout.contiguous()
            if dout.data_ptr() % 16:
                dout = dout.clone()
            n = _of_sizes('pgrf_diff_attention_backward_workspace_bytes', DTYPES[q.dtype], B, N, k.shape[1], H, k.shape[2], D, ctx.call[0])
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
            launch(q.device, 'pgrf_diff_attention_backward', _pack(q, k, v, lam, mask, None, *ctx.call, None, lse, maps, ws, n), dout.data_ptr(), ptr(dq), ptr(dk),
                   ptr(dv), ptr(dlam))
        return dq, dk if needs[1] else None, dv if needs[2] else None, dlam, None, None, None


def _check(who, q, k, v, lam, scale):
    tensor = torch.Tensor
    if not (isinstance(q, tensor) and isinstance(k, tensor) and isinstance(v, tensor) and isinstance(lam, tensor) and q.dim() == k.dim() == 5 and v.dim() == 4 and lam.dim() == 1):
        refuse(who, 'q [B, N, H, 2, d], k [B, M, Hk, 2, d], v [B, M, Hk, 2 d] and lam [H] must be tensors of these axes')
    dtype, device = q.dtype, q.device
    if dtype not in DTYPES:
        refuse(who, f'dtype {dtype} (float32, bfloat16 or float16)')
    if k.dtype != dtype or k.device != device:
        alike(who, 'k', k, dtype, device)
    if v.dtype != dtype or v.device != device:
        alike(who, 'v', v, dtype, device)
    B, N, H, two, d = q.shape
    kB, M, Hk, ktwo, kd = k.shape
    if two != 2 or d not in (32, 64, 128):
        refuse(who, f'q {tuple(q.shape)} must be [B, N, H, 2, d] with d 32, 64 or 128')
    if kB != B or ktwo != 2 or kd != d:
        refuse(who, f'k {tuple(k.shape)} must be [{B}, M, Hk, 2, {d}]')
    if v.shape != (B, M, Hk, 2 * d):
        refuse(who, f'v {tuple(v.shape)} must be [{B}, {M}, {Hk}, {2 * d}]')
    if H < 1 or Hk < 1 or H % Hk:
        refuse(who, f'{H} query heads must be a multiple of {Hk} key heads')
    if lam.shape[0] != H or lam.device != device or (lam.dtype != dtype and lam.dtype != torch.float32):
        refuse(who, f'lam must be [{H}] on {device}, float32 or of the type of q')
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        refuse(who, 'scale must be positive')
    return scale


def diff_attention(q, k, v, lam, *, causal=False, key_mask=None, scale=None):
    """q [B, N, H, 2, d], k [B, M, Hk, 2, d], v [B, M, Hk, 2 d], lam [H] -> [B, N, H, 2 d].

    float32, bfloat16 or float16 (lam of that type or float32); d 32, 64 or 128; H a multiple of Hk: the query heads h Hk/H share a key head.  Any strides (rows
    that do not start at multiples of 16 bytes are copied first).  key_mask [B, M] bool, False: no query sees the key, and what it holds does not matter.
    causal: query i sees keys up to i + M - N, so the last query stands at the last key.  A query that sees no key gives 0 and
    has no part in any gradient, whatever it and its gradient hold.  scale: 1/sqrt(d) unless given.
    Sizes: B Hk below 2^25, B H N and, with gradients, B Hk M below 2^29 fit the launches; what does not fit is refused.  M up to 2^30, H 2 d up to 2^22.
    Softmax and sums are float.  Probabilities are not rounded to fewer bits than the output holds where 32 queries or 64 keys at most share a key head, and in bfloat16
    from 1024 such queries and B H N M d = 2^33 on; elsewhere they are, each map's by itself, to the tensors' type for the product with v, as are the maps' difference and the
    score gradients in the backward pass (in float16 brought into its range first).  Gradients (first derivatives, by backward) to
    q, k, v and lam; they do not depend on scheduling."""
    who = 'diff_attention'
    scale = _check(who, q, k, v, lam, scale)
    if key_mask is not None:
        require(torch.is_tensor(key_mask) and key_mask.dtype == torch.bool and key_mask.device == q.device and tuple(key_mask.shape) == tuple(k.shape[:2]), who,
                f'key_mask must be a bool tensor {list(k.shape[:2])} on {q.device}')
    no_tangents(who, q, k, v, lam)
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
    lengths[b] - N + i.  N = 1 is the step of a served model.  The lengths are read on the device, so a captured step follows them.  Probabilities
    are rounded where diff_attention's are: not where 32 query heads and tokens at most share a key head.  No gradients."""
    who = 'diff_attention_cached'
    scale = _check(who, q, k_cache, v_cache, lam, scale)
    if not (isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int32 and lengths.device == q.device and lengths.dim() == 1 and lengths.shape[0] == q.shape[0]):
        refuse(who, f'lengths must be an int32 tensor [{q.shape[0]}] on {q.device}')
    if (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or lam.requires_grad) and torch.is_grad_enabled():
        refuse(who, 'no gradients over a cache: call it under torch.no_grad(), or diff_attention with a key_mask')
    no_tangents(who, q, k_cache, v_cache, lam)
    on_gpu(q, who)
    return _forward(_aligned(q), _aligned(k_cache), _aligned(v_cache), lam.contiguous(), None, lengths.contiguous(), True, scale, False)[0]
