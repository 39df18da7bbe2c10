"""Rotary positions (csrc/rotary.hip): pair i of a head's first channels turns by position * f_i, so that the products of two heads see the
difference of their positions.  Positions may be whole (tokens) or continuous (the depths of a ray's samples)."""
import torch

from ._token import DTYPES, ROTARY, alike, first_derivatives_only, launch, no_tangents, on_gpu, refuse, require

_SCALINGS = {None: 0, 'linear': 1, 'ntk': 2, 'parts': 3}             # PGRF_ROTARY_* of include/panogrf_hip.h
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}
_MAX_DIM = 256


def _heads(t):
    """[B, N, ..., D] as [B, N, heads, D] with the channels side by side."""
    d = t.dim()
    if d != 4:
        t = t.flatten(2, -2) if d > 4 else t.unsqueeze(2)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _launch(q, k, positions, call, backward):
    """-> tensors of the shapes of q and k, contiguous."""
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    B, N = q.shape[:2]
    if B and N:
        rot, interleaved, base, scaling, factor, trained, low, high, magnitude = call
        q4 = _heads(q)
        qs, hq, D = q4.stride(), q4.shape[2], q4.shape[3]
        if k is None:
            kp, kop, ks, hk = 0, 0, (0, 0, 0), 0
        else:
            k4 = _heads(k)
            kp, kop, ks, hk = k4.data_ptr(), k_out.data_ptr(), k4.stride(), k4.shape[2]
        launch(q.device, 'pgrf_rotary', ROTARY.pack(q4.data_ptr(), kp, positions.data_ptr(), q_out.data_ptr(), kop, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
                                                    N if positions.dim() == 2 and B > 1 else 0, base, factor, trained, low, high, DTYPES[q.dtype], B, N, D, hq, hk,
                                                    rot, interleaved, _POSITIONS[positions.dtype], scaling, backward, magnitude))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, call):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.call = call
        return _launch(q, k, positions, call, 0)

    @staticmethod
    @first_derivatives_only
    def backward(ctx, dq, dk):
        positions, = ctx.saved_tensors
        needs = ctx.needs_input_grad
        if not needs[0]:
            dq = None
        if not needs[1]:
            dk = None
        if dq is None:
            return None, None if dk is None else _launch(dk, None, positions, ctx.call, 1)[0], None, None
        return (*_launch(dq, dk, positions, ctx.call, 1), None, None)


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
    and `magnitude` multiplies every turned pair.  float32, bfloat16 or float16; gradients to q and k by backward (positions
    have none)."""
    who = 'rotary'
    require(isinstance(q, torch.Tensor) and q.dim() >= 3, who, 'q must be [B, N, ..., D]')
    dtype, device, shape = q.dtype, q.device, q.shape
    if dtype not in DTYPES:
        refuse(who, f'dtype {dtype} (float32, bfloat16 or float16)')
    B, N, D = shape[0], shape[1], shape[-1]
    if k is not None:
        if not isinstance(k, torch.Tensor) or k.dtype != dtype or k.device != device:
            alike(who, 'k', k, dtype, device)
        require(k.dim() >= 3 and k.shape[:2] == shape[:2] and k.shape[-1] == D, who, 'k must be [B, N, ..., D] with the axes of q')
        require(k.numel() > 0 or B * N == 0, who, 'k has no heads')
    rot = D if rotary_dim is None else int(rotary_dim)
    if not 2 <= rot <= min(D, _MAX_DIM) or rot % 2:
        refuse(who, f'rotary_dim {rot} (even, at most {min(D, _MAX_DIM)})')
    if layout != 'half' and layout != 'interleaved':
        refuse(who, f"layout {layout!r} ('half' or 'interleaved')")
    if scaling not in _SCALINGS:
        refuse(who, f"scaling {scaling!r} (None, 'linear', 'ntk' or 'parts')")
    require(isinstance(positions, torch.Tensor) and positions.dtype in _POSITIONS and positions.device == device, who,
            'positions must be an int32, int64, float32 or float64 tensor on the device of q')
    if positions.shape != shape[1:2] and positions.shape != shape[:2]:
        refuse(who, f'positions {tuple(positions.shape)} must be [{N}] or [{B}, {N}]')
    require(q.numel() > 0 or B * N == 0, who, 'q has no heads')
    if positions.requires_grad and torch.is_grad_enabled():
        refuse(who, 'positions have no gradient: detach them')
    no_tangents(who, q, k, positions)
    on_gpu(q, who)
    call = (rot, int(layout == 'interleaved'), float(base), _SCALINGS[scaling], float(factor), float(trained_length), float(low), float(high),
            float(magnitude))
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        return _Rotary.apply(q, k, positions, call)
    return _launch(q, k, positions, call, 0)
