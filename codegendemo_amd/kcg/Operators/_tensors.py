"""What the operators on torch tensors share: type codes, checks that name the argument, the stream of a call."""
import torch

from ... import _native
from ..Utils import EnumKernelDType

CODE = {torch.float8_e4m3fn: int(EnumKernelDType.float8), torch.float16: int(EnumKernelDType.float16),
        torch.bfloat16: int(EnumKernelDType.bfloat16), torch.float32: int(EnumKernelDType.float32)}
GROUP = 128
E4M3 = torch.float8_e4m3fn
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def groups(n):
    return -(-n // GROUP)


def stream_of(device_index):
    """torch's current stream of the device, as the raw handle the library takes."""
    if _current_stream is not None:
        return _current_stream(device_index)
    return torch.cuda.current_stream(device_index).cuda_stream


def check(status):
    if status < 0:
        _native.check(status)


def matrix(name, t, rows, cols, dtype, device):
    """A [rows, cols] tensor of `dtype` on `device` whose rows are contiguous; returns its row stride."""
    if t.dtype is dtype and t.device == device and t.shape == (rows, cols):
        s = t.stride()
        if s[1] == 1 or cols <= 1:
            return s[0]
        raise ValueError(f"{name}: the elements of a row must lie side by side, got strides {s}")
    refuse(name, t, rows, cols, dtype, device)


def strides2(name, t, rows, cols, device):
    """A float32 [rows, cols] tensor of any strides; returns them."""
    if t.dtype is torch.float32 and t.device == device and t.shape == (rows, cols):
        return t.stride()
    refuse(name, t, rows, cols, torch.float32, device)


def refuse(name, t, rows, cols, dtype, device):
    if t.dtype is not dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    raise ValueError(f"{name} must have shape ({rows}, {cols}), got {tuple(t.shape)}")


def on_gpu(name, t):
    """The device of the tensor, which has to be a GPU; no operator has another path."""
    if not t.is_cuda:
        raise TypeError(f"{name} must be on a GPU, got {t.device}: the operators have no CPU path")
    return t.device


# Outputs an operator makes itself: known strides, so they pass by the checks.  A small call is over sooner on the GPU than
# on the host, where making an output by torch.empty and slicing it would cost as much as all of the checks.

def new_e4m3(rows, cols, device):
    """An e4m3 matrix whose rows start on 16 bytes, and its row stride."""
    ld = -(-cols // 16) * 16
    return torch.empty_strided((rows, cols), (ld, 1), dtype=E4M3, device=device), ld


def new_matrix(rows, cols, dtype, device):
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)
