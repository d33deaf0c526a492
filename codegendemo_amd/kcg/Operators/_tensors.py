"""What the experts' layer needs of torch tensors: type codes, checks that name the argument, the stream of a call.  (The small
operators have the same in csrc/kcg_torch.cc: their calls are over sooner on the GPU than such checks in Python.)"""
import torch

from ... import _native
from ..Utils import EnumKernelDType

CODE = {torch.float8_e4m3fn: int(EnumKernelDType.float8), torch.float16: int(EnumKernelDType.float16),
        torch.bfloat16: int(EnumKernelDType.bfloat16), torch.float32: int(EnumKernelDType.float32)}
GROUP = 128
E4M3 = torch.float8_e4m3fn


def groups(n):
    return -(-n // GROUP)


def stream_of(device_index):
    """torch's current stream of the device, as the raw handle the library takes."""
    return torch.cuda.current_stream(device_index).cuda_stream


def check(status):
    if status < 0:
        _native.check(status)


def matrix(name, t, rows, cols, dtype, device):
    """A [rows, cols] tensor of `dtype` on `device` whose rows are contiguous; returns its row stride."""
    if t.dtype is not dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must have shape ({rows}, {cols}), got {tuple(t.shape)}")
    s = t.stride()
    if s[1] != 1 and cols > 1:
        raise ValueError(f"{name}: the elements of a row must lie side by side, got strides {s}")
    return s[0]


def on_gpu(name, t):
    """The device of the tensor, which has to be a GPU; no operator has another path."""
    if not t.is_cuda:
        raise TypeError(f"{name} must be on a GPU, got {t.device}: the operators have no CPU path")
    return t.device
