"""Matrix product of e4m3 operands with a scale for each block of 128, beside the tuned products of Operators.matmul: sizes are
run-time arguments (a serving program's row count changes from call to call), so nothing is compiled or tuned per size."""
import torch

from ... import _native_ops
from ._tensors import CODE, E4M3, check, groups, matrix, new_matrix, on_gpu, stream_of, strides2


def matmul_fp8(a, a_scale, b, b_scale, out=None, out_dtype=torch.bfloat16):
    """out[m, n] = sum over groups g of 128: a_scale[m, g] * b_scale[n // 128, g] * sum over k in g of a[m, k] * b[n, k].

    a            [M, K] e4m3, a_scale [M, ceil(K / 128)] float32: what rmsnorm_quant and swiglu_quant return
    b            [N, K] e4m3 (a weight as it is stored), b_scale [ceil(N / 128), ceil(K / 128)] float32
    out          [M, N] bfloat16, float16 or float32 (default: a new tensor of out_dtype); rows contiguous, any row stride
    Rows of a and b start on 16 bytes (K itself is free); the scales have any strides.  Sums are held in float32 and rounded
    once.  Runs on torch's current stream of the tensors' device."""
    device = on_gpu("a", a)
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError(f"a and b must be matrices, got shapes {tuple(a.shape)} and {tuple(b.shape)}")
    (m, k), n = a.shape, b.shape[0]
    a_s = matrix("a", a, m, k, E4M3, device)
    b_s = matrix("b", b, n, k, E4M3, device)
    g = groups(k)
    as_m, as_g = strides2("a_scale", a_scale, m, g, device)
    bs_n, bs_g = strides2("b_scale", b_scale, groups(n), g, device)
    if out is not None:
        out_dtype = out.dtype
    code = CODE.get(out_dtype)
    if code is None or out_dtype is E4M3:
        raise TypeError(f"out must be bfloat16, float16 or float32, got {out_dtype}")
    if out is None:
        out, o_s = new_matrix(m, n, out_dtype, device), n
    else:
        o_s = matrix("out", out, m, n, out_dtype, device)
    if m and n:
        check(_native_ops.lib().kcg_matmul_fp8(
            _native_ops.MATMUL_FP8.pack(a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), out.data_ptr(), a_s, as_m, as_g, b_s, bs_n,
                                        bs_g, o_s, m, n, k, code), device.index, stream_of(device.index)))
    return out
