/*
 * kcg_ops.h — the operators of the 8-bit serving path in libkcg_gemm.so: the norm and the activation that make e4m3
 * operands, the product of such operands, and a layer of routed experts for a few tokens.
 *
 * Same conventions as kcg_gemm.h: plain C, device addresses as integers, 0 or a negative kcg_status, the text of a failure
 * in kcg_last_error(), asynchronous on the caller's stream, no device memory allocated, nothing thrown.  Unlike the
 * tuned products of kcg_gemm.h nothing is compiled per size: the kernels take their sizes at run time and lie ready in the
 * library (built for gfx950).  The reference has no counterpart of these operators (its float8 type code,
 * include/Common/Utils.h:110-120, names a type that no kernel of it uses).
 *
 * 8-bit values: OCP e4m3 ("float8_e4m3fn": largest 448, no infinity).  A scale (float32) belongs to 128 consecutive values
 * of a row, counted from the row's start, or for a weight to a block of 128 rows x 128 columns; the last group of a row (the
 * last block) may be shorter.  A value stands for value * scale.
 *
 * Rows of 8-bit operands start on 16 bytes: base addresses and row strides are multiples of 16 (the row length is not
 * bound: what lies between its end and the next multiple of 16 is not written, and when read does not count, whatever it
 * holds).  Strides are in elements.  Outputs overlap neither inputs nor each other where nothing else is said.  `device` is the
 * device the memory and the stream belong to; the calling thread's current device is the same before and after.
 *
 * The first call on a device loads the library's code object there, which must not happen inside a stream capture: call
 * kcg_ops_load (or the operator once) before.  Afterwards every call can be captured into a HIP graph.
 */
#ifndef KCG_OPS_H
#define KCG_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* type code of e4m3 operands, beside kcg_dtype (16 and 32-bit types: KCG_DT_FLOAT16, KCG_DT_BFLOAT16, KCG_DT_FLOAT32) */
enum { KCG_DT_E4M3 = 1 };

/* Loads the operators' kernels on `device`. */
int kcg_ops_load(int device);

/* r = x + residual (float32 sum; r = x without one), residual_out = r rounded to x's type,
 * y = r / sqrt(mean(r^2) + eps) * weight, and y in e4m3: scale = max(max|y|, 1e-10) / 448 per 128 values,
 * q = y / scale rounded to nearest even.  A row that holds NaN or infinity gives NaN scales where they arise, as the
 * formula does.  residual_out may be residual itself (in place); y may be 0 (not wanted). */
typedef struct kcg_rmsnorm_quant_args {
  int64_t x, residual, residual_out; /* [rows, cols] of `dtype`; residual and residual_out both 0: no addition */
  int64_t weight;                    /* [cols] of `weight_dtype`: dtype or KCG_DT_FLOAT32 */
  int64_t y;                         /* [rows, cols] of `dtype`, or 0 */
  int64_t q, scale;                  /* [rows, cols] e4m3, [rows, ceil(cols / 128)] float32 */
  int64_t x_stride, residual_stride, residual_out_stride, y_stride, q_stride; /* from row to row */
  int64_t scale_stride_row, scale_stride_group;
  int64_t rows, cols, dtype, weight_dtype;
  double eps;
} kcg_rmsnorm_quant_args;
int kcg_rmsnorm_quant(const kcg_rmsnorm_quant_args* args, int device, uint64_t stream);

/* h = gate / (1 + exp(-gate)) * up in e4m3 with scales as above; gate = columns [0, cols) of a row of gate_up, up = columns
 * [cols, 2 cols). */
typedef struct kcg_swiglu_quant_args {
  int64_t gate_up; /* [rows, 2 cols] of `dtype` */
  int64_t q, scale;
  int64_t gate_up_stride, q_stride, scale_stride_row, scale_stride_group;
  int64_t rows, cols, dtype;
} kcg_swiglu_quant_args;
int kcg_swiglu_quant(const kcg_swiglu_quant_args* args, int device, uint64_t stream);

/* c[m, n] = sum_g a_scale[m, g] b_scale[n / 128, g] sum_{k in g} a[m, k] b[n, k], rounded once to c_dtype
 * (KCG_DT_BFLOAT16, KCG_DT_FLOAT16, KCG_DT_FLOAT32).
 * float32 results: all sums in float32.  16-bit results: the 8-bit matrix instruction adds the products of 8 neighbouring k (8 i ..
 * 8 i + 7) on a common exponent and drops of each what is below 2^-13 of the largest; sums over these in float32.  A result may so be off
 * by 2^-10 sum |a_scale b_scale a b| beside its rounding: 1.4e-5 of it on normal data, but possibly all of it where large products cancel
 * each other.  A caller that needs such sums takes float32 results. */
typedef struct kcg_matmul_fp8_args {
  int64_t a, a_scale; /* [m, k] e4m3, [m, ceil(k / 128)] */
  int64_t b, b_scale; /* [n, k] e4m3, [ceil(n / 128), ceil(k / 128)] */
  int64_t c;          /* [m, n] */
  int64_t a_stride, a_scale_stride_row, a_scale_stride_group;
  int64_t b_stride, b_scale_stride_row, b_scale_stride_group;
  int64_t c_stride;
  int64_t m, n, k, c_dtype;
} kcg_matmul_fp8_args;
int kcg_matmul_fp8(const kcg_matmul_fp8_args* args, int device, uint64_t stream);
/* Name of the kernel that a product of these sizes runs (as a profiler shows it; "" for an empty one); needs no GPU.  Writes
 * at most out_len bytes with the closing 0 and returns the name's length, or a negative status. */
int kcg_matmul_fp8_kernel(int64_t m, int64_t n, int64_t k, int64_t c_dtype, char* out, int out_len);

/* A layer of routed experts for at most 64 tokens: the topk largest logits of a token (equal ones: the lower index) choose
 * its experts, p = softmax over them (renormalize) or over all experts,
 *   h_e = silu(W1_e x) * (W3_e x),   out = sum_e p_e W2_e h_e,
 * W1 the first `inter` rows of w13[e], W3 the others; sums in float32, h kept in 16 significant bits (two bfloat16 numbers).  A logit of
 * -infinity takes an expert out: if it is among the topk all the same its weight is 0 and it adds nothing; a token with no other logits
 * gets zeros.
 * weight_dtype KCG_DT_E4M3 (block scales; dtype KCG_DT_BFLOAT16 or KCG_DT_FLOAT16) or KCG_DT_BFLOAT16 (dtype the same).
 * hidden and inter are multiples of 16; experts <= 512, topk <= 16.
 * workspace: kcg_moe_workspace_bytes() bytes on 16, in use until the stream has passed the call. */
typedef struct kcg_moe_layer_args {
  int64_t x, logits;       /* [tokens, hidden] of `dtype`, [tokens, experts] float32 */
  int64_t w13, w13_scale;  /* [experts, 2 inter, hidden], [experts, ceil(2 inter / 128), ceil(hidden / 128)] contiguous */
  int64_t w2, w2_scale;    /* [experts, hidden, inter], [experts, ceil(hidden / 128), ceil(inter / 128)] contiguous */
  int64_t out;             /* [tokens, hidden] of `dtype` */
  int64_t ids, probs;      /* out: [tokens, topk] contiguous, int32 and float32, by falling logit */
  int64_t workspace, workspace_bytes;
  int64_t x_stride, logits_stride, out_stride;
  int64_t w13_stride_expert, w13_stride_row, w2_stride_expert, w2_stride_row; /* multiples of 16 bytes */
  int64_t tokens, experts, topk, hidden, inter, dtype, weight_dtype, renormalize;
} kcg_moe_layer_args;
int kcg_moe_layer(const kcg_moe_layer_args* args, int device, uint64_t stream);
/* Bytes of a call's workspace, or KCG_ERR_ARGUMENT for sizes that kcg_moe_layer refuses. */
int64_t kcg_moe_workspace_bytes(int64_t tokens, int64_t experts, int64_t topk, int64_t hidden, int64_t inter);

#ifdef __cplusplus
}
#endif
#endif /* KCG_OPS_H */
