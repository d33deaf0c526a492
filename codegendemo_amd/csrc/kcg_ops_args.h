// kcg_ops_args.h — the argument blocks of the operators' kernels, one definition for the host and the device side.
#pragma once
#include <stdint.h>

namespace kcg_ops {

struct NormArgs {
  const void* x;
  const void* residual;      // may be null
  void* residual_out;        // null exactly if residual is
  const void* weight;
  void* y;                   // may be null
  uint8_t* q;
  float* scale;
  int64_t x_stride, residual_stride, residual_out_stride, y_stride, q_stride, scale_stride_t, scale_stride_g;
  int rows, cols;
  int weight_f32;            // the weight is in 32 bits although x is not
  float eps;
};

struct SwigluArgs {
  const void* gate_up;
  uint8_t* q;
  float* scale;
  int64_t in_stride, q_stride, scale_stride_t, scale_stride_g;
  unsigned rows;
  int cols;                  // I: gate = columns [0, I), up = [I, 2 I)
};

struct MatmulArgs {
  const uint8_t* a;          // [M, K] e4m3
  const uint8_t* b;          // [N, K] e4m3
  const float* sa;           // [M, ceil(K / 128)]
  const float* sb;           // [ceil(N / 128), ceil(K / 128)]
  void* c;                   // [M, N]
  int64_t lda, ldb, ldc, sa_m, sa_k, sb_n, sb_k;
  int M, N, K, KB;           // KB = ceil(K / 128)
  int c_wide;                // rows of C take 4-element stores
  int grid_m, grid_n;        // tiles (tile kernel)
};

constexpr int SKINNY_WAVES = 8;

constexpr int MOE_T = 64;        // most tokens of a call of the experts' layer
constexpr int MOE_E = 512;       // most experts
constexpr int MOE_K = 16;        // most experts of a token
constexpr int MOE_ITEMS = 640;   // most runs of up to 8 tokens of one expert: one per expert, and T k / 8 more
constexpr int UP_WAVES = 8;
constexpr int DOWN_WAVES = 16;
constexpr int MOE_FEW = 4;             // most tokens of the second kernel for few tokens, and most bytes of h that it keeps in LDS
constexpr int MOE_H_LDS = 128 * 1024;
constexpr int DOWN_MANY_WAVES = 8;
constexpr int DOWN_MANY_COLS = 64;     // columns of out a block of the second kernel for more tokens makes

struct MoeArgs {
  const void* x;               // [T, H]
  const float* logits;         // [T, E]
  const void* w13;             // [E, 2 I, H]
  const void* w2;              // [E, H, I]
  const float* s13;            // [E, ceil(2 I / 128), ceil(H / 128)], 8-bit weights only
  const float* s2;             // [E, ceil(H / 128), ceil(I / 128)]
  void* out;                   // [T, H]
  int32_t* ids;                // [T, k] out: the chosen experts, by falling logit
  float* probs;                // [T, k] out: their weights
  void* h_hi;                  // workspace: [T k, I] twice
  void* h_lo;
  float* picked;               // workspace: [T, k] logits of the chosen (renormalised) or their probabilities
  int* parts;                  // workspace: how many parts of I there are
  float* y;                    // workspace: [parts, T, k, H] products, to be weighed and added
  int64_t x_stride, logits_stride, out_stride;
  int64_t w13_e, w13_r, w2_e, w2_r;     // elements from expert to expert, row to row
  int T, E, k, H, I, slots;
  int renormalize;
  int split;                   // first kernel: waves that share 16 rows (>= 2)
  int max_parts;               // second kernel for more tokens: most parts of I that y has room for
};

}  // namespace kcg_ops
