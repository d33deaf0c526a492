// kcg_ops_quant.h — the two operators that make 8-bit operands: root-mean-square norm with the residual's addition, and the
// gated activation.  Both are bound by memory: one pass, 16-byte accesses, the row in registers between the sum and its use.
// Measured: norm with residual and y, 8192 x 4096 bf16, 55.7 us (5.44 TB/s; a copy reaches 5.06); one row 2.6 us, which is
// a launch and two latencies; activation, 4096 x 8192 bf16, 31.8 us (5.3 TB/s), 16 x 4096 2.6 us.
#pragma once
#include "kcg_ops_common.h"

namespace kcg_ops {

// r = x + residual, y = r / sqrt(mean r^2 + eps) * weight.  NT threads share a row (NT = 64: four rows a block, no
// barrier), each holds VPT vectors of 8 elements in registers between the sum of squares and its use; VPT = 0: the row
// does not fit and is read (and added) a second time.  A group of 128 is the 16 lanes of a DPP row, so its maximum
// costs four DPP instructions.
template <class T, int NT, int VPT>
__device__ void norm_kernel(const NormArgs& a) {
  constexpr int RPB = NT == 64 ? 4 : 1;
  constexpr int NW = NT / 64;
  __shared__ float part[NW > 1 ? NW : 1];
  const int tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * RPB + (NT == 64 ? threadIdx.x >> 6 : 0);
  if (NT == 64 && row >= a.rows) return;          // (whole waves, and no barrier below)
  const int H = a.cols;
  const T* x = (const T*)a.x + row * a.x_stride;
  const T* res = a.residual ? (const T*)a.residual + row * a.residual_stride : nullptr;
  T* res_out = a.residual ? (T*)a.residual_out + row * a.residual_out_stride : nullptr;

  auto load_sum = [&](float(&r)[8], int c, bool write) {
    load8(r, x + c, H - c);
    if (res) {
      float s[8];
      load8(s, res + c, H - c);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] += s[i];
      if (write) store8(res_out + c, r, H - c);
    }
  };
  // sum of (r * pre)^2 over the row, the same in all of its threads; pre: a power of two
  constexpr int NV = VPT > 0 ? VPT : 1;
  float r[NV][8];
  auto total = [&](float pre) {
    float sum = 0.f;
    auto add = [&](const float(&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v[i] * pre, v[i] * pre, sum);
    };
    if constexpr (VPT > 0) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) add(r[v]);
    } else {
      for (int c = tid * 8; c < H; c += NT * 8) {
        load_sum(r[0], c, false);
        add(r[0]);
      }
    }
    sum = wave_sum(sum);
    if constexpr (NW > 1) {
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
      __syncthreads();
      sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) sum += part[w];
      __syncthreads();
    }
    return sum;
  };
  auto finish = [&](float(&r)[8], int c, float pre, float rstd) {
    const int n = H - c;                          // (may be <= 0: the lane still takes part in its group's maximum)
    float w[8];
    if (a.weight_f32) load8(w, (const float*)a.weight + c, n);
    else load8(w, (const T*)a.weight + c, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = i < n ? r[i] * pre * rstd * w[i] : 0.f;
    if (a.y && n > 0) store8((T*)a.y + row * a.y_stride + c, r, n);
    float scale;
    const u32x2 q = quantize_group(r, scale);
    if (n > 0) {
      store_q8(a.q + row * a.q_stride + c, q, n);
      if ((c & (GROUP - 1)) == 0) a.scale[row * a.scale_stride_t + (int64_t)(c / GROUP) * a.scale_stride_g] = scale;
    }
  };

  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * NT + tid) * 8;
      if (c < H) load_sum(r[v], c, true);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) r[v][i] = 0.f;
    }
  }
  // The squares leave float32's range where |r| passes 2^63 (or all of r is below 2^-40 and eps does not matter): such a row
  // is summed again with r scaled by a power of two, exactly.
  float pre = 1.f;
  float mean = total(1.f) / (float)H + a.eps;
  if (!(mean >= 0x1p-80f && mean < 0x1p126f)) {
    pre = mean < 1.f ? 0x1p80f : 0x1p-80f;
    mean = total(pre) / (float)H + a.eps * pre * pre;
  }
  const float rstd = 1.f / sqrtf(mean);
  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (v * NT * 8 < H) finish(r[v], (v * NT + tid) * 8, pre, rstd);
  } else {
    // whole groups of lanes run the same number of rounds: the bound is rounded up to the 16 lanes of a group
    for (int c = tid * 8; (c & ~(GROUP - 1)) < H; c += NT * 8) {
      if (c < H) load_sum(r[0], c, true);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) r[0][i] = 0.f;
      finish(r[0], c, pre, rstd);
    }
  }
}

// h = gate / (1 + exp(-gate)) * up, quantised; 16 lanes a group, a thread 8 values.  (With expf and a division, 35 vector
// instructions a value, it was bound by them: 37.5 us at 4096 x 8192, on the same card 32.4 with silu_times.)
template <class T>
__device__ void swiglu_kernel(const SwigluArgs& a) {
  const unsigned per_row = (unsigned)((a.cols + GROUP - 1) / GROUP) * 16u;
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  const unsigned row = id / per_row;
  if (row >= a.rows) return;                      // (whole groups of 16 lanes: per_row and 256 are multiples of 16)
  const int c = (int)(id - row * per_row) * 8;
  const int n = a.cols - c;
  const T* in = (const T*)a.gate_up + (int64_t)row * a.in_stride + c;
  float g[8], u[8];
  load8(g, in, n);
  load8(u, in + a.cols, n);
  float h[8];
  unsigned far = 0;                               // (as unsigned integers, negative floats lie above the others, the smallest highest)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = silu_times(g[i], u[i]);                // (behind the row: 0 times 0)
    far = max(far, __float_as_uint(g[i]));
  }
  if (far > __float_as_uint(SILU_FAR)) {          // (hardly ever: one comparison for eight values)
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = g[i] < SILU_FAR ? silu_times_far(g[i], u[i]) : h[i];
  }
  float scale;
  const u32x2 q = quantize_group(h, scale);
  if (n > 0) {
    store_q8(a.q + (int64_t)row * a.q_stride + c, q, n);
    if ((c & (GROUP - 1)) == 0) a.scale[(int64_t)row * a.scale_stride_t + (int64_t)(c / GROUP) * a.scale_stride_g] = scale;
  }
}

}  // namespace kcg_ops
