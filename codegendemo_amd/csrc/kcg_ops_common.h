// kcg_ops_common.h — what the operators of the 8-bit path share on the device: types, conversions, masked 16-byte loads, row reductions.
//
// 8-bit values are OCP e4m3 (largest 448, no infinities, NaN = 0x7f).  A scale belongs to GROUP = 128 values along a row
// (activations) or to a block of 128 x 128 (weights).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kcg_ops_args.h"

namespace kcg_ops {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// raw carriers: any element type goes through them, at any alignment the element type has
typedef u32x4 __attribute__((may_alias, aligned(2))) u32x4_u;
typedef u32x4 __attribute__((may_alias)) u32x4_a;
typedef u32x2 __attribute__((may_alias)) u32x2_a;

template <int I> struct Int {
  static constexpr int value = I;
};
// f(Int<Begin>()), ..., f(Int<End - 1>())
template <int Begin, int End, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (Begin < End) {
    f(Int<Begin>());
    static_for<Begin + 1, End>(f);
  }
}

constexpr int GROUP = 128;
constexpr float E4M3_MAX = 448.f;
constexpr float SCALE_FLOOR = 1e-10f;   // the largest magnitude of a group counts as at least this

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// 8 consecutive elements (4 to 16-byte accesses at element alignment); `n` of them exist, the others read as 0
template <class T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n) {
  T t[8];
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      typedef u32x4 __attribute__((may_alias, aligned(4))) V;
      ((V*)t)[0] = ((const V*)p)[0];
      ((V*)t)[1] = ((const V*)p)[1];
    } else {
      *(u32x4_a*)t = *(const u32x4_u*)p;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = i < n ? p[i] : (T)0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (T)v[i];   // round to nearest even
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      typedef u32x4 __attribute__((may_alias, aligned(4))) V;
      ((V*)p)[0] = ((V*)t)[0];
      ((V*)p)[1] = ((V*)t)[1];
    } else {
      *(u32x4_u*)p = *(u32x4_a*)t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = t[i];
  }
}

// Largest of the 16 lanes of a DPP row, as unsigned integers.  The bit patterns of non-negative floats order like the
// floats, and a NaN's (0x7fc00000) lies above infinity's: the maximum of magnitudes keeps a NaN, which fmaxf would drop.
__device__ __forceinline__ unsigned row_umax(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));   // row_ror:8
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));   // row_ror:4
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));   // row_ror:2
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));   // row_ror:1
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, false));
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Quantises the 8 values of each lane of a DPP row (16 lanes x 8 = one group of 128; all 16 lanes take part): the
// group's scale and this lane's 8 bytes.  The quotient is formed with the reciprocal scale 448 / amax; its rounding moves
// a value by less than 2^-22 of itself, three orders below half a step of e4m3 (2^-4).
__device__ __forceinline__ u32x2 quantize_group(const float (&v)[8], float& scale) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(row_umax(m), __float_as_uint(SCALE_FLOOR));
  const float amax = __uint_as_float(m);
  scale = amax / E4M3_MAX;
  const float inv = E4M3_MAX / amax;
  float t[8];
  // (not finite: infinity over infinity and the like are NaN in e4m3, which has no infinities)
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = v[i] * inv;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], hi, true);
  return u32x2{(unsigned)lo, (unsigned)hi};
}

// g / (1 + exp(-g)) * up to 8 half steps of float32, g not below SILU_FAR, in two
// transcendental and nine other instructions; expf and a division take some thirty.  exp(-g) = 2^p (1 + lo ln 2), where lo is
// what the rounding of p = -g log2(e) left out (times |g| otherwise, which is what expf reduces its argument against).
// The maximum keeps the factor positive, and not NaN where p is infinite: g = infinity gives infinity.  NaN stays NaN through p.
constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596299e-8f, LN2 = 0.693147182f;
__device__ __forceinline__ float silu_times(float g, float up) {
  const float p = g * -LOG2E;
  const float lo = fmaf(g, -LOG2E_REST, fmaf(g, -LOG2E, -p));
  const float den = fmaf(__builtin_amdgcn_exp2f(p), fmaxf(fmaf(lo, LN2, 1.f), .5f), 1.f);
  return g * __builtin_amdgcn_rcpf(den) * up;
}
// The same below SILU_FAR, where 1 + exp(-g) is exp(-g): its reciprocal leaves the normal numbers at g = -87.3, while times a large
// `up` the product does not.  So exp(g) is made 2^96 times too large (96 - p is exact: p lies in [115, 2^24) or is so large that
// the power is 0) and the product is put right at the end.  To 6 half steps down to g = -154, 0 behind it, where |g exp(g) up| is
// below 1e-26 for any `up`; g = -infinity gives NaN, as infinity times 0 does.
constexpr float SILU_FAR = -80.f;
__device__ __forceinline__ float silu_times_far(float g, float up) {
  const float p = g * -LOG2E;
  const float lo = fmaf(g, -LOG2E_REST, fmaf(g, -LOG2E, -p));
  const float e = __builtin_amdgcn_exp2f(96.f - p) * fmaxf(fmaf(lo, -LN2, 1.f), .5f);
  return g * e * up * 0x1p-96f;
}

// 8 bytes of a quantised row whose start is 16-byte aligned; bytes behind the row's end stay as they were
__device__ __forceinline__ void store_q8(uint8_t* p, u32x2 q, int n) {
  if (n >= 8) {
    *(u32x2_a*)p = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)((i < 4 ? q[0] : q[1]) >> (8 * (i & 3)));
  }
}

// 16 bytes at p + k of a row of K bytes: what lies at or behind K reads as zero and is not touched beyond the 16-byte
// chunk that holds K - 1 (rows start on 16 bytes and are 16 bytes apart at least)
__device__ __forceinline__ u32x4 load16_masked(const uint8_t* p, int k, int K) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k < K) {
    v = *(const u32x4_a*)(p + k);
    const int n = K - k;
    if (n < 16) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int left = n - 4 * w;
        v[w] = left >= 4 ? v[w] : left <= 0 ? 0u : v[w] & (0xffffffffu >> (32 - 8 * left));
      }
    }
  }
  return v;
}

__device__ __forceinline__ i32x8 join(u32x4 a, u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// ---- 16 x 16 x 32 products on 16-bit operands, and e4m3 values as such ----------------------------------
struct Bf16Ops {
  typedef bf16x8 vec;
  static __device__ __forceinline__ f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ vec widen(unsigned q0, unsigned q1) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, 1.0f, true);
    return vec{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
struct F16Ops {
  typedef f16x8 vec;
  static __device__ __forceinline__ f32x4 mma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ vec widen(unsigned q0, unsigned q1) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q0, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q0, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q1, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q1, 1.0f, true);
    return vec{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};

// D[16 x 16] = A[16 x 128] B[128 x 16] on e4m3.  Lane l holds 32 bytes of row (column) l % 16; which 32 of the 128 k
// values is the same function of l / 16 for both operands, so any split of the 128 into four parts serves.  D: lane l
// holds rows 4 (l / 16) .. + 3 of column l % 16.
//
// Two ways.  E4m3Dot: one 8-bit instruction.  It adds the products of 8 neighbouring k values on a common exponent and
// drops what lies more than 13 bits below the largest of them (measured: 2^3 beside 2^16 is kept, 2^2 is lost; the 16 x 16 x 32
// form does the same): at most 2^-10 of the sum of the magnitudes, 1.4e-5 of the result on normal data, where a 16-bit result's half step
// is larger (bf16 2^-8, fp16 2^-11); where products cancel it may be all of the result, and it is above what a float32 result
// promises.  WideDot: the same values as bf16, which holds them exactly, in four instructions of half the rate, with float32
// sums.  Results in 16 bits take the first, for its rate (4096^3: 65 us, on the same card in float32 130), in 32 bits the second.
struct E4m3Dot {
  typedef i32x8 frag;
  static __device__ __forceinline__ frag make(i32x8 q) { return q; }
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b) {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 0, 0, 0, 0, 0, 0);
  }
};
struct WideDot {
  struct frag {
    bf16x8 v[4];
  };
  static __device__ __forceinline__ frag make(i32x8 q) {
    frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = Bf16Ops::widen((unsigned)q[2 * i], (unsigned)q[2 * i + 1]);
    return f;
  }
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b) {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = Bf16Ops::mma(a.v[i], b.v[i], d);
    return d;
  }
};
template <class TC> struct DotOf { typedef E4m3Dot type; };
template <> struct DotOf<float> { typedef WideDot type; };

template <class T>
__device__ __forceinline__ void store4(T* p, f32x4 v, int n, bool wide) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
  if (n >= 4 && wide) {
    if constexpr (sizeof(T) == 4) *(u32x4_a*)p = *(u32x4_a*)t;
    else *(u32x2_a*)p = *(u32x2_a*)t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = t[i];
  }
}

}  // namespace kcg_ops
