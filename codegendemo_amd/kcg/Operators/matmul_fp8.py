"""Matrix product of e4m3 operands with a scale for each block of 128, beside the tuned products of Operators.matmul: sizes are
run-time arguments (a serving program's row count changes from call to call), so nothing is compiled or tuned per size."""
import torch

from ... import _native_ops


def matmul_fp8(a, a_scale, b, b_scale, out=None, out_dtype=torch.bfloat16):
    """out[m, n] = sum over groups g of 128: a_scale[m, g] * b_scale[n // 128, g] * sum over k in g of a[m, k] * b[n, k].

    a            [M, K] e4m3, a_scale [M, ceil(K / 128)] float32: what rmsnorm_quant and swiglu_quant return
    b            [N, K] e4m3 (a weight as it is stored), b_scale [ceil(N / 128), ceil(K / 128)] float32
    out          [M, N] bfloat16, float16 or float32 (default: a new tensor of out_dtype); rows contiguous, any row stride
    Rows of a and b start on 16 bytes (K itself is free); the scales have any strides.  Runs on torch's current stream of the tensors' device.

    float32 results: every sum is held in float32.  bfloat16 and float16 results come from the 8-bit matrix instruction, which adds the
    products of 8 neighbouring k on a common exponent and drops what is below 2^-13 of the largest of them, before sums in float32
    and one rounding.  That is 1.4e-5 of a result on normal data and never more than 2^-10 of the sum of the products' magnitudes; where
    large products cancel each other it can be all of the result: take float32 results there."""
    return _native_ops.torch_ops().matmul_fp8(a, a_scale, b, b_scale, out, out_dtype)
