// kcg_ops_moe.h — a layer of routed experts for a few tokens (T <= 64), in two kernels:
//   up:   h[t, j] = silu(W1_e x_t) * (W3_e x_t)           for the j-th expert e of token t
//   down: out[t]  = sum_j p[t, j] W2_e h[t, j]
// Bound by the bytes of the experts that at least one token chose: every such weight is read once, by one block, straight
// into the matrix operand.  8-bit weights become bf16 (fp16 where x is fp16) on the way, which holds e4m3 exactly; their
// block scale multiplies the fp32 sum of the 128 products that share it.  h is kept as two bf16 numbers, its rounding and
// the rounding of what is left (16 significant bits): the weights are read once either way, and the second product costs
// matrix instructions that have nothing else to do.
//
// Routing is repeated by every block of `up` instead of a kernel of its own: an expert's place among a token's logits is
// a count of larger ones, E comparisons.  Logits are compared as integers in which the order of floats is kept (ties: the
// lower index; NaN above everything), so every place 0 .. k-1 is taken exactly once whatever the logits hold.
#pragma once
#include "kcg_ops_common.h"

namespace kcg_ops {

// order of floats as order of unsigned integers; -0 counts as 0
__device__ __forceinline__ unsigned order_key(float v) {
  if (v == 0.f) return 0x80000000u;
  const unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A lane's 32 consecutive values of a group of 128 (values 32 g .. 32 g + 31 for lane l, g = l / 16) as four operands of 8.
// `n` of the 32 exist (0, 16 or 32: the extents are multiples of 16), the others are zero.
template <class Ops>
struct Frag {
  typename Ops::vec v[4];
};
template <class Ops>
__device__ __forceinline__ Frag<Ops> load_weights(const uint8_t* p, int n) {
  u32x4 a = {0u, 0u, 0u, 0u}, b = a;
  if (n > 0) a = __builtin_nontemporal_load((const u32x4_a*)p);
  if (n > 16) b = __builtin_nontemporal_load((const u32x4_a*)(p + 16));
  Frag<Ops> f;
  f.v[0] = Ops::widen(a[0], a[1]);
  f.v[1] = Ops::widen(a[2], a[3]);
  f.v[2] = Ops::widen(b[0], b[1]);
  f.v[3] = Ops::widen(b[2], b[3]);
  return f;
}
template <class Ops, class T>
__device__ __forceinline__ Frag<Ops> load_values(const T* p, int n) {
  u32x4 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = n > 8 * i ? *(const u32x4_u*)(p + 8 * i) : u32x4{0u, 0u, 0u, 0u};
  Frag<Ops> f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = __builtin_bit_cast(typename Ops::vec, t[i]);
  return f;
}
template <class Ops, class W>
__device__ __forceinline__ Frag<Ops> load_w(const W* p, int n) {
  if constexpr (sizeof(W) == 1) return load_weights<Ops>((const uint8_t*)p, n);
  else return load_values<Ops, W>(p, n);
}
template <class Ops>
__device__ __forceinline__ f32x4 mma32(const Frag<Ops>& a, const Frag<Ops>& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = Ops::mma(a.v[i], b.v[i], c);
  return c;
}
__device__ __forceinline__ void add_scaled(f32x4& acc, const f32x4& d, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = fmaf(d[i], s, acc[i]);
}

// ---- routing: which expert this block's slot serves, and for which tokens ----------------------------
struct RouteLds {
  unsigned key[MOE_E];
  int rank[MOE_T];             // the expert's place among the token's logits, -1: not chosen
  int token[MOE_T];            // the tokens that chose it, rising
  int expert, count;
};

// Slots: with T k <= E one per (token, place), the first token that chose an expert serves all of its tokens and the other
// slots of that expert stay empty; else one per expert.  Returns the number of tokens (the same in every thread).
__device__ __forceinline__ int route(const MoeArgs& a, RouteLds& s, int slot, bool designated) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int first = 0;
  if (a.slots < a.E) {
    first = slot / a.k;
    const int place = slot - first * a.k;
    const float* l = a.logits + (int64_t)first * a.logits_stride;
    unsigned mine = 0;
    if (tid < a.E) s.key[tid] = mine = order_key(l[tid]);
    __syncthreads();
    if (tid < a.E) {
      int n = 0;
      for (int e = 0; e < a.E; ++e) {
        const unsigned other = s.key[e];
        n += (other > mine || (other == mine && e < tid)) ? 1 : 0;
      }
      if (n == place) s.expert = tid;
    }
    __syncthreads();
  } else if (tid == 0) {
    s.expert = slot;
  }
  if (a.slots >= a.E) __syncthreads();
  const int ex = s.expert;
  for (int t = wave; t < a.T; t += UP_WAVES) {
    const float* l = a.logits + (int64_t)t * a.logits_stride;
    const float lex = l[ex];
    const unsigned mine = order_key(lex);
    int n = 0;
    float sum = 0.f;
    for (int e = lane; e < a.E; e += 64) {
      const float le = l[e];
      const unsigned other = order_key(le);
      n += (other > mine || (other == mine && e < ex)) ? 1 : 0;
      if (designated && !a.renormalize) sum += expf(le - lex);
    }
    // (n <= 512: nine bits a lane)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    const bool chosen = n < a.k;
    if (lane == 0) s.rank[t] = chosen ? n : -1;
    if (designated && chosen) {
      if (!a.renormalize) sum = wave_sum(sum);
      if (lane == 0) {
        const int pair = t * a.k + n;
        a.ids[pair] = ex;
        // softmax over all experts: 1 / sum exp(l' - l); an expert that is masked out (-inf) weighs nothing
        a.picked[pair] = a.renormalize ? lex : lex == -__builtin_inff() ? 0.f : 1.f / sum;
      }
    }
  }
  __syncthreads();
  if (wave == 0) {
    const bool chosen = lane < a.T && s.rank[lane] >= 0;
    const unsigned long long who = __ballot(chosen);
    if (chosen) s.token[__popcll(who & ((1ull << lane) - 1))] = lane;
    const bool again = a.slots < a.E && (who & ((1ull << first) - 1)) != 0;   // an earlier token's slot serves this expert
    const int n = again ? 0 : __popcll(who);
    if (lane == 0) s.count = n;
    if (designated) {
      int32_t* row = a.table + (int64_t)slot * MOE_SLOT;
      if (lane == 0) {
        row[0] = n;
        row[1] = ex;
      }
      if (chosen) row[2 + __popcll(who & ((1ull << lane) - 1))] = lane * a.k + s.rank[lane];
    }
  }
  __syncthreads();
  return s.count;
}

// ---- up ------------------------------------------------------------------------------------------
// grid (I / 16, slots), UP_WAVES waves: 16 gate rows and the 16 up rows beside them; the waves split H by groups of 128 and
// meet in LDS.
template <class Ops, class W, class X, int CT>
__device__ __forceinline__ void up_tiles(const MoeArgs& a, RouteLds& s, f32x4* red, int count) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int i0 = blockIdx.x * 16;
  const int ex = __builtin_amdgcn_readfirstlane(s.expert);
  const W* wg = (const W*)a.w13 + ex * a.w13_e + (int64_t)(i0 + r) * a.w13_r + g * 32;
  const W* wu = wg + (int64_t)a.I * a.w13_r;
  const int KB = (a.H + GROUP - 1) / GROUP;
  const float* sg = nullptr;
  const float* su = nullptr;
  if constexpr (sizeof(W) == 1) {
    const int rb = (2 * a.I + GROUP - 1) / GROUP;
    sg = a.s13 + ((int64_t)ex * rb + i0 / GROUP) * KB;             // (16 rows from a multiple of 16 lie in one block)
    su = a.s13 + ((int64_t)ex * rb + (a.I + i0) / GROUP) * KB;
  }
  const X* x[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) x[c] = (const X*)a.x + (int64_t)s.token[min(c * 16 + r, count - 1)] * a.x_stride + g * 32;
  f32x4 ag[CT], au[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) ag[c] = au[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](int kb, int n) {
    const Frag<Ops> fg = load_w<Ops>(wg + kb * GROUP, n), fu = load_w<Ops>(wu + kb * GROUP, n);
    float vg = 1.f, vu = 1.f;
    if constexpr (sizeof(W) == 1) {
      vg = sg[kb];
      vu = su[kb];
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const Frag<Ops> fx = load_values<Ops, X>(x[c] + kb * GROUP, n);
      if constexpr (sizeof(W) == 1) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        add_scaled(ag[c], mma32(fg, fx, z), vg);
        add_scaled(au[c], mma32(fu, fx, z), vu);
      } else {
        ag[c] = mma32(fg, fx, ag[c]);
        au[c] = mma32(fu, fx, au[c]);
      }
    }
  };
  const int full = a.H / GROUP;
  int kb = wave;
#pragma unroll 2
  for (; kb < full; kb += UP_WAVES) step(kb, 32);
  if (kb < KB) step(kb, min(32, a.H - kb * GROUP - g * 32));
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    if (c) __syncthreads();
    red[wave * 128 + lane] = ag[c];
    red[wave * 128 + 64 + lane] = au[c];
    __syncthreads();
    if (tid < 256) {
      // thread -> row tid % 16 of column tid / 16; element (row % 4) of the lane that holds it
      const int row = tid & 15, col = tid >> 4, at = (row >> 2) * 16 + col;
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int w = 0; w < UP_WAVES; ++w) {
        gate += red[w * 128 + at][row & 3];
        up += red[w * 128 + 64 + at][row & 3];
      }
      const int n = c * 16 + col;
      if (n < count) {
        const int t = s.token[n];
        const int64_t o = (int64_t)(t * a.k + s.rank[t]) * a.I + i0 + row;
        const float h = gate / (1.f + expf(-gate)) * up;
        const __bf16 hi = (__bf16)h;
        const float hf = (float)hi;
        ((__bf16*)a.h_hi)[o] = hi;
        ((__bf16*)a.h_lo)[o] = __builtin_isfinite(hf) ? (__bf16)(h - hf) : (__bf16)0.f;
      }
    }
  }
}

template <class Ops, class W, class X>
__device__ void up_kernel(const MoeArgs& a) {
  __shared__ RouteLds s;
  __shared__ f32x4 red[UP_WAVES * 128];
  const int count = route(a, s, blockIdx.y, blockIdx.x == 0);
  if (count == 0) return;
  if (count <= 16) up_tiles<Ops, W, X, 1>(a, s, red, count);
  else if (count <= 32) up_tiles<Ops, W, X, 2>(a, s, red, count);
  else up_tiles<Ops, W, X, 4>(a, s, red, count);
}

// ---- down ----------------------------------------------------------------------------------------
// grid H / 16: a block makes 16 columns of every token's row.  Work items are (expert, part of I); the waves take them in
// turn, put their partial sums side by side in LDS, and the sum over parts and places runs in a fixed order.
struct DownLds {
  int base[MOE_E + 1];         // pairs in front of an active slot
  int slot[MOE_E];             // the active slots
  int spot[MOE_T * MOE_K];     // where a pair's partial sums stand
  float prob[MOE_T * MOE_K];
  int wave_sum[2][16];
  int active;
};

template <class W, int CT>
__device__ __forceinline__ void down_item(const MoeArgs& a, const int32_t* row, int count, int base, int part, int parts, float* partial) {
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int ex = __builtin_amdgcn_readfirstlane(row[1]);
  const W* w = (const W*)a.w2 + ex * a.w2_e + (int64_t)(n0 + r) * a.w2_r + g * 32;
  const int KB = (a.I + GROUP - 1) / GROUP;
  const float* sc = nullptr;
  if constexpr (sizeof(W) == 1) sc = a.s2 + ((int64_t)ex * ((a.H + GROUP - 1) / GROUP) + n0 / GROUP) * KB;
  const __bf16* hi[CT];
  const __bf16* lo[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int64_t at = (int64_t)row[2 + min(c * 16 + r, count - 1)] * a.I + g * 32;
    hi[c] = (const __bf16*)a.h_hi + at;
    lo[c] = (const __bf16*)a.h_lo + at;
  }
  f32x4 acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](int kb, int n) {
    const Frag<Bf16Ops> fw = load_w<Bf16Ops>(w + kb * GROUP, n);
    float v = 1.f;
    if constexpr (sizeof(W) == 1) v = sc[kb];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const Frag<Bf16Ops> fh = load_values<Bf16Ops, __bf16>(hi[c] + kb * GROUP, n), fl = load_values<Bf16Ops, __bf16>(lo[c] + kb * GROUP, n);
      if constexpr (sizeof(W) == 1) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        add_scaled(acc[c], mma32(fw, fh, mma32(fw, fl, z)), v);
      } else {
        acc[c] = mma32(fw, fh, mma32(fw, fl, acc[c]));
      }
    }
  };
  const int from = KB * part / parts, to = KB * (part + 1) / parts, full = min(to, a.I / GROUP);
  int kb = from;
#pragma unroll 2
  for (; kb < full; ++kb) step(kb, 32);
  if (kb < to) step(kb, min(32, a.I - kb * GROUP - g * 32));
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int n = c * 16 + r;
    if (n < count) *(f32x4*)(partial + (((base + n) * parts + part) * 16 + g * 4)) = acc[c];
  }
}

template <class W, class X>
__device__ void down_kernel(const MoeArgs& a, float* partial) {
  __shared__ DownLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the active slots, and how many pairs lie in front of each (slots <= 512 threads)
  int n = tid < a.slots ? a.table[(int64_t)tid * MOE_SLOT] : 0;
  {
    const unsigned long long who = __ballot(n > 0);
    int before = n;                                  // inclusive sum over the wave's lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(before, d);
      before += lane >= d ? o : 0;
    }
    if (lane == 63) {
      s.wave_sum[0][wave] = __popcll(who);
      s.wave_sum[1][wave] = before;
    }
    __syncthreads();
    int at = 0, pairs = 0;
    for (int w = 0; w < wave; ++w) {
      at += s.wave_sum[0][w];
      pairs += s.wave_sum[1][w];
    }
    if (n > 0) {
      at += __popcll(who & ((1ull << lane) - 1));
      const int base = pairs + before - n;
      s.slot[at] = tid;
      s.base[at] = base;
      const int32_t* row = a.table + (int64_t)tid * MOE_SLOT + 2;
      for (int i = 0; i < n; ++i) s.spot[row[i]] = base + i;
    }
    if (tid == DOWN_WAVES * 64 - 1) s.active = at + (n > 0 ? 1 : 0);
  }
  // the weights of the pairs
  if (tid < a.T) {
    const float* l = a.picked + tid * a.k;
    if (a.renormalize) {
      const float top = l[0];                        // place 0 holds the largest
      float sum = 0.f;
      for (int j = 0; j < a.k; ++j) sum += l[j] == -__builtin_inff() ? 0.f : expf(l[j] - top);
      for (int j = 0; j < a.k; ++j) s.prob[tid * a.k + j] = l[j] == -__builtin_inff() ? 0.f : expf(l[j] - top) / sum;
    } else {
      for (int j = 0; j < a.k; ++j) s.prob[tid * a.k + j] = l[j];
    }
    if (blockIdx.x == 0)
      for (int j = 0; j < a.k; ++j) a.probs[tid * a.k + j] = s.prob[tid * a.k + j];
  }
  __syncthreads();
  const int active = s.active;
  const int KB = (a.I + GROUP - 1) / GROUP;
  const int parts = max(1, min(DOWN_WAVES / active, KB));
  for (int item = wave; item < active * parts; item += DOWN_WAVES) {
    const int at = item / parts, part = item - at * parts;
    const int32_t* row = a.table + (int64_t)s.slot[at] * MOE_SLOT;
    const int count = __builtin_amdgcn_readfirstlane(row[0]), base = s.base[at];
    if (count <= 16) down_item<W, 1>(a, row, count, base, part, parts, partial);
    else if (count <= 32) down_item<W, 2>(a, row, count, base, part, parts, partial);
    else down_item<W, 4>(a, row, count, base, part, parts, partial);
  }
  __syncthreads();
  for (int i = tid; i < a.T * 16; i += DOWN_WAVES * 64) {
    const int t = i >> 4, c = i & 15;
    float sum = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const float p = s.prob[t * a.k + j];
      const float* v = partial + (int64_t)s.spot[t * a.k + j] * parts * 16 + c;
      float y = 0.f;
      for (int q = 0; q < parts; ++q) y += v[q * 16];
      if (p != 0.f) sum = fmaf(p, y, sum);           // (a weight of 0 adds nothing, not even 0 * infinity)
    }
    ((X*)a.out)[(int64_t)t * a.out_stride + blockIdx.x * 16 + c] = (X)sum;
  }
}

}  // namespace kcg_ops
