"""Norms before and after a block, fused with the block's gate and residual scale (csrc/block_norm.hip).

A transformer block reads z, a norm of the residual stream x, and gives back y; what stands between two blocks is

    x' = x + scale * gate * Npost(y)        z' = Npre(x')

in one pass over x and y.  `kind='rms'`: N(a) = a / sqrt(mean(a^2) + eps) * w; `kind='layer'`: N(a) = (a - mean) / sqrt(var + eps) * w + b (the
form of the aggregation net's ray attention: nn.LayerNorm(16, eps=1e-6), network/ibrnet.py:160-204)."""
import torch

from ._token import BLOCK_NORM, DTYPES, alike, entry, first_derivatives_only, launch, no_tangents, on_gpu, ptr, refuse, require

_LAYER, _POST, _PRE = 1, 2, 4
_NAMES = ('x', 'y', 'gate', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')


def _launch(x, y, gate, pw, pb, qw, qb, rpg, flags, scale, eps, want_stats):
    C = x.shape[-1]
    rows = x.numel() // C
    x_out = None if y is None else torch.empty_like(x)
    z = torch.empty_like(x) if flags & _PRE else None
    stats = torch.empty(rows, 4, dtype=torch.float32, device=x.device) if want_stats else None
    if rows:
        launch(x.device, 'pgrf_block_norm', BLOCK_NORM.pack(x.data_ptr(), ptr(y), ptr(gate), ptr(pw), ptr(pb), ptr(qw), ptr(qb), ptr(x_out), ptr(z), ptr(stats),
                                                            0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, rows, rpg, DTYPES[x.dtype], C, flags, scale, eps))
    return x_out, z, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, pw, pb, qw, qb, rpg, flags, scale, eps):
        x_out, z, stats = _launch(x, y, gate, pw, pb, qw, qb, rpg, flags, scale, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, pw, pb, qw, qb, stats)
        ctx.call = (rpg, flags, scale)
        return x_out, z

    @staticmethod
    @first_derivatives_only
    def backward(ctx, dx_out, dz):
        x, y, gate, pw, pb, qw, qb, stats = ctx.saved_tensors
        rpg, flags, scale = ctx.call
        if dx_out is None and dz is None:
            return (None,) * 11
        C = x.shape[-1]
        rows = x.numel() // C
        needs = ctx.needs_input_grad
        dx, dy, dgate = (torch.empty_like(t) if need and t is not None else None for t, need in zip((x, y, gate), needs))
        columns = (pw, pb, qw, qb)
        if any(needs[3:7]):
            rooms = torch.empty(4, C, dtype=x.dtype, device=x.device).unbind(0)
            dpw, dpb, dqw, dqb = (r if need and t is not None else None for r, t, need in zip(rooms, columns, needs[3:7]))
        else:
            dpw = dpb = dqw = dqb = None
        if rows == 0:
            return tuple(None if g is None else g.zero_() for g in (dx, dy, dgate, dpw, dpb, dqw, dqb)) + (None,) * 4
        if dx_out is not None and not dx_out.is_contiguous():
            dx_out = dx_out.contiguous()
        if dz is not None and not dz.is_contiguous():
            dz = dz.contiguous()
        n, ws = 0, None                             # scratch for sums over rows: of the weights, the biases and a shared gate
        if any(needs[3:7]) or (needs[2] and rpg > 1):
            n = entry('pgrf_block_norm_backward_workspace_bytes')(rows, C, rpg)
            ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        launch(x.device, 'pgrf_block_norm_backward',
               BLOCK_NORM.pack(x.data_ptr(), ptr(y), ptr(gate), ptr(pw), ptr(pb), ptr(qw), ptr(qb), 0, 0, stats.data_ptr(), ptr(dx_out), ptr(dz), ptr(dx), ptr(dy),
                               ptr(dgate), ptr(dpw), ptr(dpb), ptr(dqw), ptr(dqb), ptr(ws), n, rows, rpg, DTYPES[x.dtype], C, flags, scale, 0.0))
        return dx, dy, dgate, dpw, dpb, dqw, dqb, None, None, None, None


def block_norm(x, y=None, gate=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, *, post=True, pre=True, kind='rms',
               scale=1.0, eps=1e-6):
    """-> (x', z) with x' = x + scale * gate * Npost(y) and z = Npre(x').

    x [..., C] (C up to 8 192) float32, bfloat16 or float16, y the same shape or None (then x' is x and only z is formed: the norm before the first
    block, or of any tensor's last axis).  gate: None (1), [C] (a layer scale), the shape of x, or x's leading axes up to some axis and then C, e.g.
    [B, C] for x [B, N, C] (one gate per sample; over 60 000 shared ones have no gradient).  All of x's type.  Weights and biases [C] or None (1 and 0); biases with kind='layer' only.  post=False leaves out
    the norm of y, pre=False the norm of x' (z is None then).  Statistics and sums are float; x' is rounded once to its type and z formed from its
    unrounded value.  All of x, y, gate, weights and biases have gradients (first derivatives, by backward;
    their sums do not depend on scheduling)."""
    who = 'block_norm'
    require(isinstance(x, torch.Tensor) and x.dim() >= 1, who, 'x must be a tensor with a channel axis')
    dtype, device, shape = x.dtype, x.device, x.shape
    if dtype not in DTYPES:
        refuse(who, f'dtype {dtype} (float32, bfloat16 or float16)')
    C = shape[-1]
    if not 1 <= C <= 8192:
        refuse(who, f'{C} channels (1 to 8192)')
    layer = kind == 'layer'
    if not layer and kind != 'rms':
        refuse(who, f"kind {kind!r} ('rms' or 'layer')")
    if y is None:
        require(gate is None, who, 'a gate needs y')
        require(pre, who, 'neither y nor a norm of x: nothing to do')
        post = False
    ts = [x, y, gate, post_weight, post_bias, pre_weight, pre_bias]
    used = (True, True, True, post, post and layer, pre, pre and layer)
    grad = False
    for i, t in enumerate(ts):
        if t is None:
            continue
        if i:
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
                alike(who, _NAMES[i], t, dtype, device)
            if i == 1 and t.shape != shape:
                refuse(who, 'y must have the shape of x')
            if i >= 3:
                if not used[i]:
                    refuse(who, f'{_NAMES[i]} has no place in this call (its norm is left out, or kind is not layer)')
                if t.dim() != 1 or t.shape[0] != C:
                    refuse(who, f'{_NAMES[i]} must have shape [{C}]')
        grad = grad or t.requires_grad
        if not t.is_contiguous():
            ts[i] = t.contiguous()
    rows = x.numel() // C
    rpg = max(rows, 1)
    if gate is not None:
        lead = gate.shape[:-1]
        require(gate.dim() >= 1 and gate.shape[-1] == C and gate.dim() <= x.dim() and lead == shape[:len(lead)], who,
                f'gate {tuple(gate.shape)} must be [C], the leading axes of x {tuple(shape)} and C, or the shape of x')
        gates = gate.numel() // C
        rpg = max(rows // max(gates, 1), 1)
        require(rpg == 1 or gates <= 60000 or not (gate.requires_grad and torch.is_grad_enabled()), who,
                'no gradient of over 60000 gate rows that are shared by several rows each: detach the gate, or expand it to the shape of x')
    no_tangents(who, *ts)
    on_gpu(x, who)
    flags = (_LAYER if layer else 0) | (_POST if post else 0) | (_PRE if pre else 0)
    if grad and torch.is_grad_enabled():
        x_out, z = _BlockNorm.apply(*ts, rpg, flags, float(scale), float(eps))
    else:
        x_out, z, _ = _launch(*ts, rpg, flags, float(scale), float(eps), False)
    return (x if x_out is None else x_out), z
