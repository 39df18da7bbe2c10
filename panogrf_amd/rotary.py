"""Rotary positions (csrc/rotary.hip): pair i of a head's first channels turns by position * f_i, so that the products of two heads see the
difference of their positions.  Positions may be whole (tokens) or continuous (the depths of a ray's samples)."""
import torch

from ._lib import lib
from ._token import alike, dtype_code, on_device, on_gpu, require

_SCALINGS = {None: 0, 'linear': 1, 'ntk': 2, 'parts': 3}             # PGRF_ROTARY_* of include/panogrf_hip.h
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}
_MAX_DIM = 256


def _launch(q, k, positions, call, backward):
    """q, k [B,N,heads,D], any strides with the channels side by side."""
    B, N, hq, D = q.shape
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if B and N:
        rot, interleaved, base, scaling, factor, trained, low, high, magnitude = call
        qs, ks = q.stride(), (0, 0, 0) if k is None else k.stride()
        with on_device(q.device) as stream:
            lib.check(lib.pgrf_rotary(q.data_ptr(), qs[0], qs[1], qs[2], hq, None if k is None else k.data_ptr(), ks[0], ks[1], ks[2],
                                      0 if k is None else k.shape[2], positions.data_ptr(), _POSITIONS[positions.dtype],
                                      N if positions.dim() == 2 and B > 1 else 0, dtype_code(q, 'rotary'), B, N, D, rot, interleaved, base, scaling,
                                      factor, trained, low, high, magnitude, backward, q_out.data_ptr(), None if k is None else k_out.data_ptr(), stream))
    return q_out, k_out


def _rows(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, call):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.call = call
        return _launch(q, k, positions, call, 0)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, = ctx.saved_tensors
        needs = ctx.needs_input_grad
        gs = [g if need else None for g, need in ((dq, needs[0]), (dk, needs[1]))]
        first, second = (gs[0], gs[1]) if gs[0] is not None else (gs[1], None)
        if first is None:
            return None, None, None, None
        a, b = _launch(_rows(first), None if second is None else _rows(second), positions, ctx.call, 1)
        return (a, b, None, None) if gs[0] is not None else (None, a, None, None)


def rotary(q, k, positions, *, rotary_dim=None, layout='half', base=10000.0, scaling=None, factor=1.0, trained_length=4096, low=1.0, high=32.0,
           magnitude=1.0):
    """-> (q', k'): q [B, N, ..., D] and k [B, N, ..., D] (or None) with their first `rotary_dim` channels (None: all; even, up to 256) turned.

    Axes between the tokens and the channels are heads (a pair of maps [.., H, 2, d] counts as 2 H).  layout 'half': pairs (i, i + rotary_dim/2),
    'interleaved': (2i, 2i + 1).  positions [N] or [B, N]: int32, int64, float32 or float64, any size: angles are formed and reduced in 64 bits.
    f_i = base^(-2i/rotary_dim); for contexts longer than the trained one `scaling` makes that
      'linear'  f_i / factor
      'ntk'     with base * factor^(rotary_dim/(rotary_dim-2))
      'parts'   f_i (t + (1-t)/factor), t = clamp((trained_length f_i/2pi - low)/(high - low), 0, 1): pairs of over `high` turns in the trained
                context stay, those of under `low` are stretched
    and `magnitude` multiplies every turned pair.  float32, bfloat16 or float16; gradients to q and k."""
    who = 'rotary'
    require(torch.is_tensor(q) and q.dim() >= 3, who, 'q must be [B, N, ..., D]')
    dtype_code(q, who)
    alike(who, q.dtype, q.device, k=k)
    B, N, D = q.shape[0], q.shape[1], q.shape[-1]
    require(k is None or (k.dim() >= 3 and k.shape[:2] == q.shape[:2] and k.shape[-1] == D), who, 'k must be [B, N, ..., D] with the axes of q')
    rot = D if rotary_dim is None else int(rotary_dim)
    require(2 <= rot <= min(D, _MAX_DIM) and rot % 2 == 0, who, f'rotary_dim {rot} (even, at most {min(D, _MAX_DIM)})')
    require(layout in ('half', 'interleaved'), who, f"layout {layout!r} ('half' or 'interleaved')")
    require(scaling in _SCALINGS, who, f"scaling {scaling!r} (None, 'linear', 'ntk' or 'parts')")
    require(torch.is_tensor(positions) and positions.device == q.device and positions.dtype in _POSITIONS, who,
            'positions must be an int32, int64, float32 or float64 tensor on the device of q')
    require(tuple(positions.shape) in ((N,), (B, N)), who, f'positions {tuple(positions.shape)} must be [{N}] or [{B}, {N}]')
    require(q.numel() > 0 or B * N == 0, who, 'q has no heads')
    require(k is None or k.numel() > 0 or B * N == 0, who, 'k has no heads')
    on_gpu(q, who)
    call = (rot, int(layout == 'interleaved'), float(base), _SCALINGS[scaling], float(factor), float(trained_length), float(low), float(high),
            float(magnitude))
    q4, k4 = (None if t is None else _rows(t.flatten(2, -2) if t.dim() > 3 else t.unsqueeze(2)) for t in (q, k))
    positions = positions.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        q_out, k_out = _Rotary.apply(q4, k4, positions, call)
    else:
        q_out, k_out = _launch(q4, k4, positions, call, 0)
    return q_out.view(q.shape), None if k is None else k_out.view(k.shape)
