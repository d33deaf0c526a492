"""ctypes binding of the operators of the 8-bit path in libkcg_gemm.so (C ABI: include/kcg_ops.h).

A call's arguments travel as one packed block (all fields are 64 bits wide), which costs a launch about a microsecond of
host time where a ctypes argument for each field would cost several."""
import ctypes
import struct

from . import _native

EXPORTS = ("kcg_ops_load", "kcg_rmsnorm_quant", "kcg_swiglu_quant", "kcg_matmul_fp8", "kcg_matmul_fp8_kernel", "kcg_moe_layer", "kcg_moe_workspace_bytes")
DT_E4M3 = 1
RMSNORM_QUANT = struct.Struct("=18qd")      # kcg_rmsnorm_quant_args
SWIGLU_QUANT = struct.Struct("=10q")        # kcg_swiglu_quant_args
MATMUL_FP8 = struct.Struct("=16q")          # kcg_matmul_fp8_args
MOE_LAYER = struct.Struct("=26q")           # kcg_moe_layer_args

_ops = None


def lib():
    """The library with the operators' signatures set."""
    global _ops
    if _ops is None:
        L = _native.lib()
        for name in EXPORTS:
            if not hasattr(L, name):
                raise ImportError(f"{_native.LIB_PATH} has no {name}: build it again (__graft_entry__.build())")
        for name in ("kcg_rmsnorm_quant", "kcg_swiglu_quant", "kcg_matmul_fp8", "kcg_moe_layer"):
            getattr(L, name).argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_uint64]
        L.kcg_moe_workspace_bytes.argtypes = [ctypes.c_int64] * 5
        L.kcg_moe_workspace_bytes.restype = ctypes.c_int64
        L.kcg_matmul_fp8_kernel.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_char_p, ctypes.c_int]
        L.kcg_ops_load.argtypes = [ctypes.c_int]
        _ops = L
    return _ops


def load(device=0):
    """Loads the operators' kernels on a device (otherwise the first call there does; not inside a stream capture)."""
    _native.check(lib().kcg_ops_load(int(device)))


def moe_workspace_bytes(tokens, experts, topk, hidden, inter):
    return _native.check(lib().kcg_moe_workspace_bytes(tokens, experts, topk, hidden, inter))


def matmul_fp8_kernel(m, n, k, c_dtype):
    """Name of the kernel that a product of these sizes runs (c_dtype: a code of EnumKernelDType)."""
    buf = ctypes.create_string_buffer(256)
    _native.check(lib().kcg_matmul_fp8_kernel(m, n, k, int(c_dtype), buf, len(buf)))
    return buf.value.decode()
