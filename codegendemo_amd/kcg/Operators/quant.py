"""Operators that make the 8-bit operands of matmul_fp8: the norm in front of a product and the gated activation between two.

Values are OCP e4m3 with a float32 scale for each 128 of a row: scale = max(max|v|, 1e-10) / 448, q = v / scale rounded to
nearest even.  Both run on torch's current stream of the tensors' device; the formulas and limits stand in include/kcg_ops.h."""
import torch

from ... import _native_ops
from ._tensors import CODE, E4M3, check, groups, matrix, new_e4m3, new_matrix, on_gpu, stream_of, strides2


def rmsnorm_quant(x, weight, eps=1e-6, residual=None, residual_out=None, q=None, scale=None, y=None, want_y=False):
    """Root-mean-square norm of the rows of x (plus residual) in e4m3: -> (q, scale, y, residual_out).

    x            [T, H] bfloat16, float16 or float32; rows contiguous, any row stride
    weight       [H], x's type or float32
    residual     [T, H] of x's type: r = x + residual is what is normed (the float32 sum, not its rounding);
                 r rounded to x's type goes to residual_out (default: a new tensor; pass residual itself for in place)
    q, scale     [T, H] e4m3 whose rows start on 16 bytes, [T, ceil(H / 128)] float32 of any strides (default: new ones)
    y            [T, H] of x's type: the normed row in 16 (32) bits too, for what reads it unquantised, such as a router;
                 written if it is given or want_y is set, else None is returned"""
    device = on_gpu("x", x)
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, got shape {tuple(x.shape)}")
    dtype = x.dtype
    if dtype not in CODE or dtype is E4M3:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {dtype}")
    t, h = x.shape
    x_s = matrix("x", x, t, h, dtype, device)
    if weight.shape != (h,) or (h > 1 and weight.stride(0) != 1) or weight.device != device or weight.dtype not in (dtype, torch.float32):
        raise ValueError(f"weight must be a contiguous vector of {h} values of {dtype} or torch.float32 on {device}")
    r_p = ro_p = r_s = ro_s = 0
    if residual is not None:
        r_s = matrix("residual", residual, t, h, dtype, device)
        if residual_out is None:
            residual_out, ro_s = new_matrix(t, h, dtype, device), h
        else:
            ro_s = matrix("residual_out", residual_out, t, h, dtype, device)
        r_p, ro_p = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    if q is None:
        q, q_s = new_e4m3(t, h, device)
    else:
        q_s = matrix("q", q, t, h, E4M3, device)
    s_t, s_g = groups(h), 1
    if scale is None:
        scale = new_matrix(t, s_t, torch.float32, device)
    else:
        s_t, s_g = strides2("scale", scale, t, s_t, device)
    y_p = y_s = 0
    if y is not None:
        y_p, y_s = y.data_ptr(), matrix("y", y, t, h, dtype, device)
    elif want_y:
        y, y_s = new_matrix(t, h, dtype, device), h
        y_p = y.data_ptr()
    code = CODE[dtype]
    if t and h:
        check(_native_ops.lib().kcg_rmsnorm_quant(
            _native_ops.RMSNORM_QUANT.pack(x.data_ptr(), r_p, ro_p, weight.data_ptr(), y_p, q.data_ptr(), scale.data_ptr(), x_s, r_s, ro_s, y_s, q_s,
                                           s_t, s_g, t, h, code, CODE[weight.dtype], eps), device.index, stream_of(device.index)))
    return q, scale, y, residual_out


def swiglu_quant(gate_up, q=None, scale=None):
    """silu(gate) * up in e4m3: -> (q, scale).

    gate_up      [T, 2 I] bfloat16, float16 or float32: gate = the first I columns, up = the others (what one product with
                 the two weights stacked gives); rows contiguous, any row stride
    q, scale     [T, I] e4m3 whose rows start on 16 bytes, [T, ceil(I / 128)] float32 of any strides (default: new ones)"""
    device = on_gpu("gate_up", gate_up)
    if gate_up.dim() != 2 or gate_up.shape[1] % 2:
        raise ValueError(f"gate_up must be a matrix with an even number of columns, got shape {tuple(gate_up.shape)}")
    dtype = gate_up.dtype
    if dtype not in CODE or dtype is E4M3:
        raise TypeError(f"gate_up must be bfloat16, float16 or float32, got {dtype}")
    t, i = gate_up.shape[0], gate_up.shape[1] // 2
    in_s = matrix("gate_up", gate_up, t, 2 * i, dtype, device)
    if q is None:
        q, q_s = new_e4m3(t, i, device)
    else:
        q_s = matrix("q", q, t, i, E4M3, device)
    s_t, s_g = groups(i), 1
    if scale is None:
        scale = new_matrix(t, s_t, torch.float32, device)
    else:
        s_t, s_g = strides2("scale", scale, t, s_t, device)
    if t and i:
        check(_native_ops.lib().kcg_swiglu_quant(
            _native_ops.SWIGLU_QUANT.pack(gate_up.data_ptr(), q.data_ptr(), scale.data_ptr(), in_s, q_s, s_t, s_g, t, i, CODE[dtype]),
            device.index, stream_of(device.index)))
    return q, scale
