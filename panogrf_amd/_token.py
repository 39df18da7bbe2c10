"""What the token operators (block_norm, rotary, attention) share: checks of their tensors and the launch's device and stream."""
import torch

from ._lib import PgrfError

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # PGRF_DTYPE_* of include/panogrf_hip.h


def dtype_code(t, who):
    try:
        return DTYPES[t.dtype]
    except KeyError:
        raise PgrfError(f'{who}: dtype {t.dtype} (float32, bfloat16 or float16)') from None


def require(ok, who, what):
    if not ok:
        raise PgrfError(f'{who}: {what}')


def on_gpu(t, who):
    if not t.is_cuda:
        raise PgrfError(f'{who}: the tensors must be on a ROCm GPU (gfx950); there is no CPU fallback')


def alike(who, dtype, device, **tensors):
    """Every tensor given has this dtype and device."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise PgrfError(f'{who}: {name} must be a tensor')
        if t.device != device:
            raise PgrfError(f'{who}: {name} is on {t.device}, expected {device}')
        if t.dtype != dtype:
            raise PgrfError(f'{who}: {name} is {t.dtype}, expected {dtype}')


class on_device:
    """The launch goes to the tensors' device, whatever the current one is, and to that device's current stream."""
    __slots__ = ('index', 'before')

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)
        return False


def ptr(t):
    return None if t is None else t.data_ptr()
