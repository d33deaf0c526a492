// kcg_ops.hip — the kernels of the 8-bit path, as the host side (kcg_ops.cc) names them.  Built for gfx950 into one code
// object that libkcg_gemm.so carries; sizes are run-time arguments, so a handful of instantiations serves every call.
#include "kcg_ops_matmul.h"
#include "kcg_ops_moe.h"
#include "kcg_ops_quant.h"

using namespace kcg_ops;

#define NORM(T, NAME, NT, VPT)                                                                       \
  extern "C" __global__ void __launch_bounds__(NT == 64 ? 256 : NT) kcg_norm_##NAME##_##NT##_##VPT(NormArgs a) { norm_kernel<T, NT, VPT>(a); }
#define NORMS(T, NAME) \
  NORM(T, NAME, 64, 1) NORM(T, NAME, 128, 1) NORM(T, NAME, 256, 1) NORM(T, NAME, 512, 1) NORM(T, NAME, 1024, 1) NORM(T, NAME, 1024, 2) NORM(T, NAME, 1024, 0)
NORMS(__bf16, bf16)
NORMS(_Float16, f16)
NORMS(float, f32)

#define SWIGLU(T, NAME) \
  extern "C" __global__ void __launch_bounds__(256) kcg_swiglu_##NAME(SwigluArgs a) { swiglu_kernel<T>(a); }
SWIGLU(__bf16, bf16)
SWIGLU(_Float16, f16)
SWIGLU(float, f32)

#define SKINNY(TC, NAME, CT, RT)                                                                              \
  extern "C" __global__ void __launch_bounds__(SKINNY_WAVES * 64) kcg_mm8_skinny_##NAME##_##CT##x##RT(MatmulArgs a) { \
    __shared__ f32x4 red[SKINNY_WAVES * CT * RT * 64];                                                         \
    skinny_kernel<TC, CT, RT, SKINNY_WAVES>(a, red);                                                           \
  }
#define SKINNIES(TC, NAME) SKINNY(TC, NAME, 1, 1) SKINNY(TC, NAME, 1, 2) SKINNY(TC, NAME, 2, 1) SKINNY(TC, NAME, 2, 2)
// BM x BN tile, WM x WN waves a group, S stages, KS groups; W: waves per SIMD the registers have to leave room for
#define TILE(TC, NAME, BM, BN, WM, WN, S, KS, W)                                                                              \
  extern "C" __global__ void __launch_bounds__(WM * WN * KS * 64, W) kcg_mm8_tile_##NAME##_##BM##x##BN##_##WM##x##WN##x##KS(   \
      MatmulArgs a) {                                                                                                         \
    __shared__ __attribute__((aligned(1024))) uint8_t smem[TilePlan<BM, BN, WM, WN, S, KS>::LDS];                             \
    tile_kernel<TC, BM, BN, WM, WN, S, KS>(a, smem);                                                                          \
  }
#define MATMULS(TC, NAME)                                                                                                     \
  SKINNIES(TC, NAME)                                                                                                          \
  TILE(TC, NAME, 32, 32, 2, 1, 4, 4, 2) TILE(TC, NAME, 64, 32, 4, 1, 4, 2, 2) TILE(TC, NAME, 64, 64, 2, 2, 4, 1, 2)           \
  TILE(TC, NAME, 64, 64, 2, 2, 4, 2, 2) TILE(TC, NAME, 64, 128, 2, 2, 2, 1, 2)                                                \
  TILE(TC, NAME, 128, 128, 2, 2, 2, 1, 2)
MATMULS(__bf16, bf16)
MATMULS(_Float16, f16)
MATMULS(float, f32)
TILE(__bf16, bf16, 128, 64, 4, 2, 4, 1, 2) TILE(__bf16, bf16, 128, 128, 4, 2, 4, 1, 2) TILE(__bf16, bf16, 256, 256, 4, 2, 2, 1, 2)
TILE(_Float16, f16, 128, 64, 4, 2, 4, 1, 2) TILE(_Float16, f16, 128, 128, 4, 2, 4, 1, 2) TILE(_Float16, f16, 256, 256, 4, 2, 2, 1, 2)

#define MOE(OPS, W, X, NAME)                                                                                        \
  extern "C" __global__ void __launch_bounds__(UP_WAVES * 64, 4) kcg_moe_up_##NAME(MoeArgs a) { up_kernel<OPS, W, X>(a); } \
  extern "C" __global__ void __launch_bounds__(DOWN_WAVES * 64) kcg_moe_down_few_##NAME(MoeArgs a) {               \
    extern __shared__ __attribute__((aligned(16))) float partial[];                                                 \
    down_few_kernel<W, X>(a, partial);                                                                              \
  }
MOE(Bf16Ops, uint8_t, __bf16, e4m3_bf16)
MOE(F16Ops, uint8_t, _Float16, e4m3_f16)
MOE(Bf16Ops, __bf16, __bf16, bf16_bf16)
// (these keep nothing in x's type)
#define DOWN_MANY(W, NAME, PER) \
  extern "C" __global__ void __launch_bounds__(DOWN_MANY_WAVES * 64, 2) kcg_moe_down_many_##NAME##_##PER(MoeArgs a) { down_many_kernel<W, PER>(a); }
DOWN_MANY(uint8_t, e4m3, 8) DOWN_MANY(uint8_t, e4m3, 16)
DOWN_MANY(__bf16, bf16, 8) DOWN_MANY(__bf16, bf16, 16)
extern "C" __global__ void __launch_bounds__(256) kcg_moe_combine_bf16(MoeArgs a) { combine_kernel<__bf16>(a); }
extern "C" __global__ void __launch_bounds__(256) kcg_moe_combine_f16(MoeArgs a) { combine_kernel<_Float16>(a); }
