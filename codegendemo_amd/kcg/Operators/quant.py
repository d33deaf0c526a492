"""Operators that make the 8-bit operands of matmul_fp8: the norm in front of a product and the gated activation between two.

Values are OCP e4m3 with a float32 scale for each 128 of a row: scale = max(max|v|, 1e-10) / 448, q = v / scale rounded to
nearest even.  Both run on torch's current stream of the tensors' device; the formulas and limits stand in include/kcg_ops.h."""
from ... import _native_ops


def rmsnorm_quant(x, weight, eps=1e-6, residual=None, residual_out=None, q=None, scale=None, y=None, want_y=False):
    """Root-mean-square norm of the rows of x (plus residual) in e4m3: -> (q, scale, y, residual_out).

    x            [T, H] bfloat16, float16 or float32; rows contiguous, any row stride
    weight       [H], x's type or float32
    residual     [T, H] of x's type: r = x + residual is what is normed (the float32 sum, not its rounding);
                 r rounded to x's type goes to residual_out (default: a new tensor; pass residual itself for in place)
    q, scale     [T, H] e4m3 whose rows start on 16 bytes, [T, ceil(H / 128)] float32 of any strides (default: new ones)
    y            [T, H] of x's type: the normed row in 16 (32) bits too, for what reads it unquantised, such as a router;
                 written if it is given or want_y is set, else None is returned"""
    return _native_ops.torch_ops().rmsnorm_quant(x, weight, eps, residual, residual_out, q, scale, y, want_y)


def swiglu_quant(gate_up, q=None, scale=None):
    """silu(gate) * up in e4m3: -> (q, scale).

    gate_up      [T, 2 I] bfloat16, float16 or float32: gate = the first I columns, up = the others (what one product with
                 the two weights stacked gives); rows contiguous, any row stride
    q, scale     [T, I] e4m3 whose rows start on 16 bytes, [T, ceil(I / 128)] float32 of any strides (default: new ones)"""
    return _native_ops.torch_ops().swiglu_quant(gate_up, q, scale)
