"""Norms before and after a block, fused with the block's gate and residual scale (csrc/block_norm.hip).

A transformer block reads z, a norm of the residual stream x, and gives back y; what stands between two blocks is

    x' = x + scale * gate * Npost(y)        z' = Npre(x')

in one pass over x and y.  `kind='rms'`: N(a) = a / sqrt(mean(a^2) + eps) * w; `kind='layer'`: N(a) = (a - mean) / sqrt(var + eps) * w + b (the
form of the aggregation net's ray attention: nn.LayerNorm(16, eps=1e-6), network/ibrnet.py:160-204)."""
import torch

from ._lib import PgrfError, lib
from ._token import alike, dtype_code, on_device, on_gpu, ptr, require

_LAYER, _POST, _PRE = 1, 2, 4


def _launch(x, y, gate, rpg, pw, pb, qw, qb, flags, scale, eps, want_stats):
    C = x.shape[-1]
    rows = x.numel() // C
    x_out = torch.empty_like(x) if y is not None else None
    z = torch.empty_like(x) if flags & _PRE else None
    stats = torch.empty(rows, 4, dtype=torch.float32, device=x.device) if want_stats else None
    if rows:
        with on_device(x.device) as stream:
            lib.check(lib.pgrf_block_norm(x.data_ptr(), ptr(y), ptr(gate), rpg, ptr(pw), ptr(pb), ptr(qw), ptr(qb), dtype_code(x, 'block_norm'), rows, C,
                                          flags, scale, eps, ptr(x_out), ptr(z), ptr(stats), stream))
    return x_out, z, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, pw, pb, qw, qb, rpg, flags, scale, eps):
        x_out, z, stats = _launch(x, y, gate, rpg, pw, pb, qw, qb, flags, scale, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, pw, pb, qw, qb, stats)
        ctx.call = (rpg, flags, scale)
        return x_out, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dx_out, dz):
        x, y, gate, pw, pb, qw, qb, stats = ctx.saved_tensors
        rpg, flags, scale = ctx.call
        if dx_out is None and dz is None:
            return (None,) * 11
        C = x.shape[-1]
        rows = x.numel() // C
        needs = ctx.needs_input_grad
        new = lambda i, t: torch.empty_like(t) if t is not None and needs[i] else None
        dx, dy, dgate, dpw, dpb, dqw, dqb = (new(i, t) for i, t in enumerate((x, y, gate, pw, pb, qw, qb)))
        if rows == 0:
            return tuple(None if g is None else g.zero_() for g in (dx, dy, dgate, dpw, dpb, dqw, dqb)) + (None,) * 4
        dx_out, dz = (None if g is None else g.contiguous() for g in (dx_out, dz))
        with on_device(x.device) as stream:
            n = lib.pgrf_block_norm_backward_workspace_bytes(rows, C, rpg)
            ws = torch.empty(n, dtype=torch.uint8, device=x.device)
            lib.check(lib.pgrf_block_norm_backward(x.data_ptr(), ptr(y), ptr(gate), rpg, ptr(pw), ptr(pb), ptr(qw), stats.data_ptr(), ptr(dx_out),
                                                   ptr(dz), dtype_code(x, 'block_norm'), rows, C, flags, scale, ptr(dx), ptr(dy), ptr(dgate),
                                                   ptr(dpw), ptr(dpb), ptr(dqw), ptr(dqb), ws.data_ptr(), n, stream))
        return dx, dy, dgate, dpw, dpb, dqw, dqb, None, None, None, None


def block_norm(x, y=None, gate=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, *, post=True, pre=True, kind='rms',
               scale=1.0, eps=1e-6):
    """-> (x', z) with x' = x + scale * gate * Npost(y) and z = Npre(x').

    x [..., C] (C up to 8 192) float32, bfloat16 or float16, y the same shape or None (then x' is x and only z is formed: the norm before the first
    block, or of any tensor's last axis).  gate: None (1), [C] (a layer scale), the shape of x, or x's leading axes up to some axis and then C, e.g.
    [B, C] for x [B, N, C] (one gate per sample).  Weights and biases [C] or None (1 and 0); biases with kind='layer' only.  post=False leaves out
    the norm of y, pre=False the norm of x' (z is None then).  Statistics and sums are float; x' is rounded once to its type and z formed from its
    unrounded value.  All of x, y, gate, weights and biases have gradients (first derivatives; their sums do not depend on scheduling)."""
    who = 'block_norm'
    require(torch.is_tensor(x) and x.dim() >= 1, who, 'x must be a tensor with a channel axis')
    dtype_code(x, who)
    C = x.shape[-1]
    require(1 <= C <= 8192, who, f'{C} channels (1 to 8192)')
    require(kind in ('rms', 'layer'), who, f"kind {kind!r} ('rms' or 'layer')")
    require(y is not None or gate is None, who, 'a gate needs y')
    require(y is not None or pre, who, 'neither y nor a norm of x: nothing to do')
    alike(who, x.dtype, x.device, y=y, gate=gate, post_weight=post_weight, post_bias=post_bias, pre_weight=pre_weight, pre_bias=pre_bias)
    require(y is None or y.shape == x.shape, who, 'y must have the shape of x')
    post = bool(post) and y is not None
    for name, t, used in (('post_weight', post_weight, post), ('post_bias', post_bias, post and kind == 'layer'), ('pre_weight', pre_weight, pre),
                          ('pre_bias', pre_bias, pre and kind == 'layer')):
        require(t is None or used, who, f'{name} has no place in this call (its norm is left out, or kind is not layer)')
        require(t is None or tuple(t.shape) == (C,), who, f'{name} must have shape [{C}]')
    rows = x.numel() // C
    rpg = max(rows, 1)
    if gate is not None:
        lead = tuple(gate.shape[:-1])
        require(gate.dim() >= 1 and gate.shape[-1] == C and lead == tuple(x.shape[:len(lead)]) and gate.dim() <= x.dim(), who,
                f'gate {tuple(gate.shape)} must be [C], the leading axes of x {tuple(x.shape)} and C, or the shape of x')
        rpg = max(rows // max(gate.numel() // C, 1), 1)
        require(rpg == 1 or rpg >= rows or gate.numel() // C <= 60000, who, 'over 60000 gate rows that are shared by several rows each')
    flags = (_LAYER if kind == 'layer' else 0) | (_POST if post else 0) | (_PRE if pre else 0)
    on_gpu(x, who)
    ts = [None if t is None else t.contiguous() for t in (x, y, gate, post_weight, post_bias, pre_weight, pre_bias)]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        x_out, z = _BlockNorm.apply(*ts, rpg, flags, float(scale), float(eps))
    else:
        x_out, z, _ = _launch(ts[0], ts[1], ts[2], rpg, *ts[3:], flags, float(scale), float(eps), False)
    return (x if x_out is None else x_out), z
