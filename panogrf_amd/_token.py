"""What the token operators (block_norm, rotary, attention) share: checks of their tensors and the call into the library.

A small call costs the host more than the GPU, so the way down is short: argument structures are packed as bytes in one go, entry points are looked up once,
and the device is switched only where the tensors are on another one."""
import struct

import torch
from torch.autograd import forward_ad

from ._lib import PgrfError, lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # PGRF_DTYPE_* of include/panogrf_hip.h

# the structures of include/panogrf_hip.h, field by field
BLOCK_NORM = struct.Struct('@20PN2q3i2f4x')
ROTARY = struct.Struct('@5P7q5d11if')
DIFF_ATTN = struct.Struct('@10PN12q9if')

_entries = {}


def entry(name):
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(lib, name)
    return f


def refuse(who, what):
    raise PgrfError(f'{who}: {what}')


def dtype_code(t, who):
    code = DTYPES.get(t.dtype)
    if code is None:
        refuse(who, f'dtype {t.dtype} (float32, bfloat16 or float16)')
    return code


def require(ok, who, what):
    if not ok:
        raise PgrfError(f'{who}: {what}')


def on_gpu(t, who):
    if not t.is_cuda:
        refuse(who, 'the tensors must be on a ROCm GPU (gfx950); there is no CPU fallback')


def alike(who, name, t, dtype, device):
    """The tensor has this dtype and device."""
    if not isinstance(t, torch.Tensor):
        refuse(who, f'{name} must be a tensor')
    if t.device != device:
        refuse(who, f'{name} is on {t.device}, expected {device}')
    if t.dtype != dtype:
        refuse(who, f'{name} is {t.dtype}, expected {dtype}')


def no_tangents(who, *tensors):
    """No tensor carries a tangent of forward-mode differentiation, which the outputs would lose.  (_current_level: -1 outside of it, as nearly always; asking each
    tensor costs more than all other checks.)"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                refuse(who, 'no forward-mode derivatives (dual tensors, torch.func.jvp): use backward')


def launch(device, name, *args):
    """Calls an entry point with `args` and the current stream of the tensors' device, whatever the current device is."""
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = entry(name)(*args, torch.cuda.current_stream(index).cuda_stream)
    else:
        rc = entry(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        lib.check(rc)


def first_derivatives_only(backward):
    """torch's once_differentiable where a graph of the gradients is asked for (its wrapper costs more than a small backward pass)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        no_tangents('backward', *grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


def ptr(t):
    return 0 if t is None else t.data_ptr()
