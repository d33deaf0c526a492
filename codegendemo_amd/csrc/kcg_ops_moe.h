// kcg_ops_moe.h — a layer of routed experts for a few tokens (T <= 64), in two kernels, or three:
//   up:   h[t, j] = silu(W1_e x_t) * (W3_e x_t)           for the j-th expert e of token t
//   down: out[t]  = sum_j p[t, j] W2_e h[t, j]            one kernel for a few tokens, else products and their sum apart
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

// order of floats as order of unsigned integers; -0 counts as 0; 0 is below every key
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned u = __float_as_uint(v);
  unsigned k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  if (v == 0.f) k = 0x80000000u;
  if ((u & 0x7fffffffu) > 0x7f800000u) k = 0xffffffffu;
  return k;
}

// sums over the 8 lanes of an aligned eighth of a wave
template <class T>
__device__ __forceinline__ T sum8(T v) {
  auto dpp = [](T x, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v += dpp(v, Int<0xB1>());      // quad_perm: lane ^ 1
  v += dpp(v, Int<0x4E>());      // quad_perm: lane ^ 2
  v += dpp(v, Int<0x141>());     // row_half_mirror: the other four
  return v;
}

// ---- 16-bit operands from weights and values ---------------------------------------------------------
// A group of 128 k values is four operands of 8 per lane.  Operand i of lane l (g = l / 16) holds the 8 values from
// place(g, i) on, the same for weights and values: two loads of 16 bytes cover a line of 8-bit weights.
template <class W>
__device__ __forceinline__ constexpr int place(int g, int i) {
  return sizeof(W) == 1 ? (i >> 1) * 64 + g * 16 + (i & 1) * 8 : i * 32 + g * 8;
}
template <class W> struct Raw {                       // weights as they are stored
  u32x4 v[sizeof(W) == 1 ? 2 : 4];
};
struct RawValues {
  u32x4 v[4];
};
// The loads have no branches (behind one, the compiler could not count which loads are in flight, and would wait for all of
// them): a place at or behind `n` (a multiple of 16) is read from the row's last values instead, and clear_tail() makes it zero,
// in weights and values both: either may hold an infinity there, and 0 times that is NaN.
template <class W>
__device__ __forceinline__ Raw<W> load_w(const W* row, int k, int g, int n) {
  Raw<W> q;
  constexpr int C = sizeof(W) == 1 ? 2 : 4;
#pragma unroll
  for (int i = 0; i < C; ++i) q.v[i] = *(const u32x4_a*)(row + min(k + place<W>(g, i * (4 / C)), n - 16 / (int)sizeof(W)));
  return q;
}
template <class W, class X>
__device__ __forceinline__ RawValues load_x(const X* row, int k, int g, int n) {
  RawValues q;
#pragma unroll
  for (int i = 0; i < 4; ++i) q.v[i] = *(const u32x4_u*)(row + min(k + place<W>(g, i), n - 8));
  return q;
}
template <class W>
__device__ __forceinline__ void clear_tail(Raw<W>& q, int k, int g, int n) {
  constexpr int C = sizeof(W) == 1 ? 2 : 4;
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (k + place<W>(g, i * (4 / C)) >= n) q.v[i] = u32x4{0u, 0u, 0u, 0u};
}
template <class W>
__device__ __forceinline__ void clear_tail(RawValues& q, int k, int g, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k + place<W>(g, i) >= n) q.v[i] = u32x4{0u, 0u, 0u, 0u};
}
template <class Ops, class W>
__device__ __forceinline__ typename Ops::vec operand(const Raw<W>& q, int i) {
  if constexpr (sizeof(W) == 1) return Ops::widen(q.v[i >> 1][2 * (i & 1)], q.v[i >> 1][2 * (i & 1) + 1]);
  else return __builtin_bit_cast(typename Ops::vec, q.v[i]);
}
__device__ __forceinline__ void add_scaled(f32x4& acc, const f32x4& d, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = fmaf(d[i], s, acc[i]);
}

// ---- routing: which expert this block's slot serves, and for which tokens ----------------------------
struct RouteLds {
  int rank[MOE_T];             // the expert's place among the token's logits, -1: not chosen
  int token[MOE_T];            // the tokens that chose it, rising
};

// The expert in place `place` of one token's logits (in every lane): the largest, taken out `place` times.
__device__ __forceinline__ int expert_in_place(const float* l, int E, int place) {
  const int lane = threadIdx.x & 63;
  unsigned key[MOE_E / 64];
#pragma unroll
  for (int i = 0; i < MOE_E / 64; ++i) key[i] = i * 64 + lane < E ? order_key(l[i * 64 + lane]) : 0u;
  int e = 0;
  for (int n = 0;; ++n) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < MOE_E / 64; ++i)
      if (i * 64 < E) m = max(m, key[i]);
    m = row_umax(m);
    m = max(max((unsigned)__builtin_amdgcn_readlane(m, 0), (unsigned)__builtin_amdgcn_readlane(m, 16)),
            max((unsigned)__builtin_amdgcn_readlane(m, 32), (unsigned)__builtin_amdgcn_readlane(m, 48)));
    bool found = false;
#pragma unroll
    for (int i = 0; i < MOE_E / 64; ++i)
      if (i * 64 < E && !found) {
        const unsigned long long who = __ballot(key[i] == m);
        if (who) {
          found = true;
          const int at = __ffsll(who) - 1;
          e = i * 64 + at;
          if (lane == at) key[i] = 0;
        }
      }
    if (n == place) return e;
  }
}

// Slots: with T k < E one per (token, place), the first token that chose an expert serves all of its tokens and the other
// slots of that expert stay empty; else one per expert.  Returns the number of tokens (the same in every thread).
__device__ __forceinline__ int route(const MoeArgs& a, RouteLds& s, int slot, bool designated, int& expert) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int first = 0, ex = slot;
  if (a.slots < a.E) {
    first = slot / a.k;
    ex = expert_in_place(a.logits + (int64_t)first * a.logits_stride, a.E, slot - first * a.k);
  }
  expert = ex;
  if (a.T == 1 && a.slots < a.E && (a.renormalize || !designated)) {
    // a token alone: the slot's place is all there is to know
    if (lane == 0) {
      s.rank[0] = slot;
      s.token[0] = 0;
      if (designated && wave == 0) {
        a.ids[slot] = ex;
        a.picked[slot] = a.logits[ex];
      }
    }
    __syncthreads();
    return 1;
  }
  // 8 lanes a token, 8 tokens a wave
  const int t = wave * 8 + (lane >> 3);
  if (t < a.T) {
    const float* l = a.logits + (int64_t)t * a.logits_stride;
    const float lex = l[ex];
    const unsigned mine = order_key(lex);
    const bool sums = designated && !a.renormalize;
    int n = 0;
    float sum = 0.f;
#pragma unroll 4
    for (int e = (lane & 7) * 4; e < a.E; e += 32) {
      float v[4];
      if (e + 4 <= a.E) {
        typedef f32x4 __attribute__((may_alias, aligned(4))) V;
        const f32x4 q = *(const V*)(l + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = q[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = e + i < a.E ? l[e + i] : -__builtin_inff();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned other = order_key(v[i]);
        n += e + i < a.E && (other > mine || (other == mine && e + i < ex)) ? 1 : 0;
        if (sums) sum += expf(v[i] - lex);             // (behind E: exp(-inf) = 0)
      }
    }
    n = sum8(n);
    const bool chosen = n < a.k;
    if ((lane & 7) == 0) s.rank[t] = chosen ? n : -1;
    if (designated && chosen) {
      sum = sum8(sum);
      if ((lane & 7) == 0) {
        const int pair = t * a.k + n;
        a.ids[pair] = ex;
        // softmax over all experts: 1 / sum exp(l' - l); an expert that is masked out (-inf) weighs nothing
        a.picked[pair] = a.renormalize ? lex : lex == -__builtin_inff() ? 0.f : 1.f / sum;
      }
    }
  }
  __syncthreads();
  // every wave for itself (and all write the same list)
  const int rank = lane < a.T ? s.rank[lane] : -1;
  const unsigned long long who = __ballot(rank >= 0);
  if (rank >= 0) s.token[__popcll(who & ((1ull << lane) - 1))] = lane;
  const bool again = a.slots < a.E && (who & ((1ull << first) - 1)) != 0;   // an earlier token's slot serves this expert
  return again ? 0 : __popcll(who);
}

// ---- up ------------------------------------------------------------------------------------------
// grid (x, slots), UP_WAVES waves.  A row group is 16 gate rows and the 16 up rows beside them.  `split` waves share a row
// group, each with a part of H, and meet in LDS; UP_WAVES / split row groups run side by side.  The loads of a step (a group of
// 128 of one row group) are issued before the products of the step in front of it (up to 16 tokens).  Measured: 64 tokens, 8 of 128
// experts of 1024 x 4096 in e4m3, 192 us (1.06 GB: 5.5 TB/s); a token, 8 of 64 of 1024 x 2048, 10.6 us, of which the weights' bytes are
// 5.2 and the rest a launch, the routing and the first loads, one after another.
template <class Ops, class W, class X, int CT>
__device__ __forceinline__ void up_tiles(const MoeArgs& a, RouteLds& s, f32x4* red, int ex, int count, int skip) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int split = a.split, side = UP_WAVES / split;
  const int rg_end = a.I / 16, rg = blockIdx.x * side + wave / split, part = wave % split;
  const W* wg = (const W*)a.w13 + ex * a.w13_e + (int64_t)r * a.w13_r;
  const int KB = (a.H + GROUP - 1) / GROUP, full = a.H / GROUP;
  const float* sc = sizeof(W) == 1 ? a.s13 + (int64_t)ex * ((2 * a.I + GROUP - 1) / GROUP) * KB : nullptr;
  const X* x[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) x[c] = (const X*)a.x + (int64_t)s.token[min(skip + c * 16 + r, count - 1)] * a.x_stride;
  struct Stage {
    Raw<W> g, u;
    RawValues x[CT];
    float vg, vu;
  };
  // (a row group behind the last one is computed from the last one's weights and not stored: there are barriers below)
  const int rgl = min(rg, rg_end - 1);
  const W* rowg = wg + (int64_t)rgl * 16 * a.w13_r;
  const W* rowu = rowg + (int64_t)a.I * a.w13_r;
  auto load = [&](Stage& st, int kb) {
    st.g = load_w<W>(rowg, kb * GROUP, g, a.H);
    st.u = load_w<W>(rowu, kb * GROUP, g, a.H);
#pragma unroll
    for (int c = 0; c < CT; ++c) st.x[c] = load_x<W>(x[c], kb * GROUP, g, a.H);
    if constexpr (sizeof(W) == 1) {
      // (16 rows from a multiple of 16 lie in one block of 128)
      st.vg = sc[(int64_t)(rgl * 16 / GROUP) * KB + kb];
      st.vu = sc[(int64_t)((a.I + rgl * 16) / GROUP) * KB + kb];
    }
  };
  auto write = [&](int n, int row, float gate, float up) {
    const int t = s.token[n];
    const int64_t o = (int64_t)(t * a.k + s.rank[t]) * a.I + row;
    const float h = gate < SILU_FAR ? silu_times_far(gate, up) : silu_times(gate, up);
    const __bf16 hi = (__bf16)h;
    const float hf = (float)hi;
    ((__bf16*)a.h_hi)[o] = hi;
    ((__bf16*)a.h_lo)[o] = __builtin_isfinite(hf) ? (__bf16)(h - hf) : (__bf16)0.f;
  };
  f32x4 ag[CT], au[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) ag[c] = au[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](Stage& st, int kb) {
    if (kb >= full) {
      clear_tail<W>(st.g, kb * GROUP, g, a.H);
      clear_tail<W>(st.u, kb * GROUP, g, a.H);
#pragma unroll
      for (int c = 0; c < CT; ++c) clear_tail<W>(st.x[c], kb * GROUP, g, a.H);
    }
    f32x4 dg[CT], du[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      dg[c] = sizeof(W) == 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : ag[c];
      du[c] = sizeof(W) == 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : au[c];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const typename Ops::vec fg = operand<Ops, W>(st.g, i), fu = operand<Ops, W>(st.u, i);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const typename Ops::vec fx = __builtin_bit_cast(typename Ops::vec, st.x[c].v[i]);
        dg[c] = Ops::mma(fg, fx, dg[c]);
        du[c] = Ops::mma(fu, fx, du[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      if constexpr (sizeof(W) == 1) {
        add_scaled(ag[c], dg[c], st.vg);
        add_scaled(au[c], du[c], st.vu);
      } else {
        ag[c] = dg[c];
        au[c] = du[c];
      }
    }
  };
  int kb = KB * part / split;
  const int to = KB * (part + 1) / split;
  if constexpr (CT == 1) {
    // (two named stages in turn: copying one into the other would wait for its loads)
    Stage a0, a1;
    if (kb < to) load(a0, kb);
    for (; kb + 2 < to; kb += 2) {
      load(a1, kb + 1);
      multiply(a0, kb);
      load(a0, kb + 2);
      multiply(a1, kb + 1);
    }
    if (kb + 2 == to) {
      load(a1, kb + 1);
      multiply(a0, kb);
      multiply(a1, kb + 1);
    } else if (kb < to) {
      multiply(a0, kb);
    }
  } else {
    // (two stages of two column tiles would not fit the registers of 16 waves a compute unit)
    for (; kb < to; ++kb) {
      Stage now;
      load(now, kb);
      multiply(now, kb);
    }
  }
  // the sums become h
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    __syncthreads();                              // (the sums of the tile before have been read)
    red[wave * 128 + lane] = ag[c];
    red[wave * 128 + 64 + lane] = au[c];
    __syncthreads();
    // thread -> row % 16 of column / 16 of a row group; element (row % 4) of the lane that holds it
    for (int i = tid; i < side * 256; i += UP_WAVES * 64) {
      const int q = i >> 8, row = i & 15, col = (i >> 4) & 15, at = (row >> 2) * 16 + col;
      float gate = 0.f, up = 0.f;
      for (int w = q * split; w < (q + 1) * split; ++w) {
        gate += red[w * 128 + at][row & 3];
        up += red[w * 128 + 64 + at][row & 3];
      }
      const int n = skip + c * 16 + col, to_rg = blockIdx.x * side + q;
      if (n < count && to_rg < rg_end) write(n, to_rg * 16 + row, gate, up);
    }
  }
}

// (more than 32 tokens of one expert: its weights are read once more for each further 32)
template <class Ops, class W, class X>
__device__ void up_kernel(const MoeArgs& a) {
  __shared__ RouteLds s;
  __shared__ f32x4 red[UP_WAVES * 128];
  int ex;
  const int count = route(a, s, blockIdx.y, blockIdx.x == 0, ex);
  ex = __builtin_amdgcn_readfirstlane(ex);
  for (int skip = 0; skip < count; skip += 32) {
    if (count - skip <= 16) up_tiles<Ops, W, X, 1>(a, s, red, ex, count, skip);
    else up_tiles<Ops, W, X, 2>(a, s, red, ex, count, skip);
  }
}

// ---- down ----------------------------------------------------------------------------------------
// Work items are (expert, up to 8 of its tokens): the 16 columns of a product hold the upper parts of 8 tokens' h and beside
// them the lower ones, whose sums are added at the end, so that a group of 128 costs four loads of h and not eight.  Where
// experts have more tokens an item holds 16 and takes the lower parts as a second product.  Waves take (item, part of I) in
// turn; sums over parts and over a token's places run in a fixed order.
struct SortLds {
  unsigned long long tokens[MOE_E];   // which tokens chose the expert
  int first[MOE_E];            // pairs of the experts in front of it
  short item_expert[MOE_ITEMS], item_first[MOE_ITEMS], item_count[MOE_ITEMS];   // up to 8 (16) pairs of one expert
  int pair[MOE_T * MOE_K];     // pairs (t k + place) by expert, then token
  int wave_sum[DOWN_WAVES];
  int items;
};

// The pairs in the order of their experts, cut into items; NT >= MOE_E threads, thread i has the experts of pairs i, i + NT, ...
// Ends with a barrier; at(pair, spot) is told where each pair stands.
template <int NT, int PER, class F>
__device__ __forceinline__ void sort_pairs(const MoeArgs& a, SortLds& s, const int (&expert)[MOE_T * MOE_K / NT], F&& at_spot) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pairs = a.T * a.k;
  if (a.T == 1) {
    // a token alone: its places are the items (sorting them by expert would be a fifth of the call)
    if (tid < pairs) {
      s.item_expert[tid] = (short)expert[0];
      s.item_first[tid] = s.pair[tid] = tid;
      s.item_count[tid] = 1;
      at_spot(tid, tid);
    }
    if (tid == 0) s.items = pairs;
    __syncthreads();
    return;
  }
  if (tid < a.E) s.tokens[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MOE_T * MOE_K / NT; ++i)
    if (tid + i * NT < pairs) atomicOr(&s.tokens[expert[i]], 1ull << ((tid + i * NT) / a.k));
  __syncthreads();
  // the chosen experts' items side by side, and how many pairs lie in front of each expert
  const int n = tid < a.E ? __popcll(s.tokens[tid]) : 0;
  const int mine = (n + PER - 1) / PER;            // items of this thread's expert
  int upto = n << 16 | mine;                       // inclusive sums over the wave's lanes, of pairs (<= 1024) and items (<= 512)
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    upto += lane >= d ? o : 0;
  }
  if (lane == 63) s.wave_sum[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += s.wave_sum[w];
  if (n > 0) {
    const int first = (upto >> 16) - n, at = (upto & 0xffff) - mine;
    s.first[tid] = first;
    for (int i = 0; i < mine; ++i) {
      s.item_expert[at + i] = (short)tid;
      s.item_first[at + i] = (short)(first + i * PER);
      s.item_count[at + i] = (short)min(PER, n - i * PER);
    }
  }
  if (tid == NT - 1) s.items = upto & 0xffff;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MOE_T * MOE_K / NT; ++i) {
    const int pair = tid + i * NT;
    if (pair < pairs) {
      const int spot = s.first[expert[i]] + __popcll(s.tokens[expert[i]] & ((1ull << (pair / a.k)) - 1));
      s.pair[spot] = pair;
      at_spot(pair, spot);
    }
  }
  __syncthreads();
}

// the weight of place `place` of a token, from what the first kernel picked for its k places (place 0 holds the largest logit)
__device__ __forceinline__ float pair_weight(const MoeArgs& a, const float* picked, int place) {
  const float mine = picked[place];
  if (!a.renormalize) return mine;
  const float top = picked[0];
  float sum = 0.f;
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) sum += picked[j] == -__builtin_inff() ? 0.f : expf(picked[j] - top);
  return mine == -__builtin_inff() ? 0.f : expf(mine - top) / sum;
}

// One (item, part of I) after another of a wave's share, RT tiles of 16 rows of W2 from row `n0` on beside each other.  The loads
// of a step are issued N - 1 steps before its products, across items too (named stages in turn: copying one into another
// would wait for its loads).  HL: h lies in LDS, and the loads are the weights alone.  PER: pairs of an item.
template <class W, int RT, int N, bool HL, int PER>
struct DownWave {
  struct Stage {
    Raw<W> w[RT];
    RawValues h[PER / 8];                            // (HL: read when it is used)
    const __bf16* row;
    float v;
    int kb, unit;                                    // unit: -1 - unit in its last step
  };
  const MoeArgs& a;
  const SortLds& s;
  const __bf16* h_lds;
  const int lane, r, g, KB, full, parts, units, stride, n0;
  int64_t w_row[RT];
  Stage st[N];
  f32x4 acc[RT];
  // where the loads of the wave's next step come from
  const W* w = nullptr;
  const float* sc = nullptr;
  const __bf16* h = nullptr;
  int unit, kb = 0, to = 0, left = 0;

  __device__ __forceinline__ DownWave(const MoeArgs& args, const SortLds& sort, const __bf16* hl, int row0, int part_count, int first, int step)
      : a(args), s(sort), h_lds(hl), lane(threadIdx.x & 63), r(lane & 15), g(lane >> 4), KB((a.I + GROUP - 1) / GROUP), full(a.I / GROUP),
        parts(part_count), units(sort.items * part_count), stride(step), n0(row0), unit(first) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      w_row[t] = (int64_t)min(n0 + t * 16 + r, a.H - 1) * a.w2_r;       // (rows behind the last one are not stored)
      acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int u = first; u < units; u += step) {
      const int part = u % parts;
      left += KB * (part + 1) / parts - KB * part / parts;
    }
    open();
    static_for<0, N - 1>([&](auto i_c) {
      if (decltype(i_c)::value < left) load(st[decltype(i_c)::value]);
    });
  }
  __device__ __forceinline__ void open() {
    if (unit >= units) return;
    const int which = unit / parts, part = unit - which * parts;
    const int ex = __builtin_amdgcn_readfirstlane(s.item_expert[which]), first = __builtin_amdgcn_readfirstlane(s.item_first[which]);
    const int count = __builtin_amdgcn_readfirstlane(s.item_count[which]);
    w = (const W*)a.w2 + ex * a.w2_e;
    // (RT tiles of 16 rows from a multiple of RT tiles lie in one block of 128)
    if constexpr (sizeof(W) == 1) sc = a.s2 + ((int64_t)ex * ((a.H + GROUP - 1) / GROUP) + n0 / GROUP) * KB;
    const int pair = s.pair[first + min(r & (PER - 1), count - 1)];
    if constexpr (PER == 16) h = (const __bf16*)a.h_hi + (int64_t)pair * a.I;
    else if constexpr (HL) h = h_lds + (pair + (r < 8 ? 0 : a.T * a.k)) * (a.I + 8);
    else h = (const __bf16*)(r < 8 ? a.h_hi : a.h_lo) + (int64_t)pair * a.I;
    kb = KB * part / parts;
    to = KB * (part + 1) / parts;
  }
  __device__ __forceinline__ void load(Stage& q) {
#pragma unroll
    for (int t = 0; t < RT; ++t) q.w[t] = load_w<W>(w + w_row[t], kb * GROUP, g, a.I);
    if constexpr (HL) q.row = h;
    else q.h[0] = load_x<W>(h, kb * GROUP, g, a.I);
    if constexpr (PER == 16) q.h[1] = load_x<W>(h + ((const __bf16*)a.h_lo - (const __bf16*)a.h_hi), kb * GROUP, g, a.I);
    if constexpr (sizeof(W) == 1) q.v = sc[kb];
    q.kb = kb;
    q.unit = unit;
    if (++kb == to) {
      q.unit = -1 - unit;
      unit += stride;
      open();
    }
  }
  // done(unit's item, part, sums of tile t: lane (r, g) has rows 4 g .. 4 g + 3 of the item's pair r, r < PER)
  template <class F>
  __device__ __forceinline__ void multiply(Stage& q, F&& done) {
    if constexpr (HL) q.h[0] = load_x<W>(q.row, q.kb * GROUP, g, a.I);
    if (q.kb >= full) {
#pragma unroll
      for (int t = 0; t < RT; ++t) clear_tail<W>(q.w[t], q.kb * GROUP, g, a.I);
#pragma unroll
      for (int c = 0; c < PER / 8; ++c) clear_tail<W>(q.h[c], q.kb * GROUP, g, a.I);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      f32x4 d = sizeof(W) == 1 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[t];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 f = operand<Bf16Ops, W>(q.w[t], i);
#pragma unroll
        for (int c = 0; c < PER / 8; ++c) d = Bf16Ops::mma(f, __builtin_bit_cast(bf16x8, q.h[c].v[i]), d);
      }
      if constexpr (sizeof(W) == 1) add_scaled(acc[t], d, q.v);
      else acc[t] = d;
    }
    if (q.unit < 0) {
      const int unit = -1 - q.unit, which = unit / parts;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int i = 0; i < 4 && PER == 8; ++i) acc[t][i] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(acc[t][i]), 0x128, 0xf, 0xf, false));   // row_ror:8
        done(which, unit - which * parts, t, acc[t]);
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void run(F&& done) {
    for (; left >= 2 * N - 1; left -= N) {
      static_for<0, N>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        load(st[(i + N - 1) % N]);
        multiply(st[i], done);
      });
    }
    static_for<0, 2 * N - 2>([&](auto i_c) {
      constexpr int i = decltype(i_c)::value;
      if (i + N - 1 < left) load(st[(i + N - 1) % N]);
      if (i < left) multiply(st[i % N], done);
    });
  }
};

// One token or a few whose h fits LDS: grid H / 16, a block makes 16 columns of every token's row.  The waves put their partial
// sums side by side in LDS and the block adds them up.  Four steps of loads in flight.  A token, 8 of 64 experts of 1024 x 2048:
// 8.8 us (9.0 on the card where it took 12.7 with h from memory and 11.1 with h asked for behind the sorting).
template <class W, class X>
__device__ void down_few_kernel(const MoeArgs& a, float* partial) {
  __shared__ SortLds s;
  __shared__ int spot[MOE_FEW * MOE_K];              // where a pair stands in the order of experts
  __shared__ float picked[MOE_FEW * MOE_K], prob[MOE_FEW * MOE_K];
  constexpr int NT = DOWN_WAVES * 64;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pairs = a.T * a.k;                       // (at most as many as threads; experts at most half of that)
  const int expert[1] = {tid < pairs ? a.ids[tid] : 0};
  const float my_value = tid < pairs ? a.picked[tid] : 0.f;
  // LDS behind the partial sums: h, upper parts, then lower ones, rows 8 values longer than they are (other banks).  The
  // workspace holds the two planes side by side, pairs * I values each (I a multiple of 16): copied 16 bytes at a time.
  constexpr int H_CHUNKS = MOE_H_LDS / 16 / NT;
  const int per_row = a.I / 8, chunks = 2 * pairs * per_row, h_row = a.I + 8;
  u32x4 hv[H_CHUNKS];
#pragma unroll
  for (int i = 0; i < H_CHUNKS; ++i) hv[i] = ((const u32x4_a*)a.h_hi)[min(tid + i * NT, chunks - 1)];
  if (tid < pairs) picked[tid] = my_value;
  sort_pairs<NT, 8>(a, s, expert, [&](int pair, int at) { spot[pair] = at; });
  const int parts = max(1, min(DOWN_WAVES / s.items, (a.I + GROUP - 1) / GROUP));
  __bf16* h_lds = (__bf16*)(partial + pairs * parts * 16);
  DownWave<W, 1, 4, true, 8> d(a, s, h_lds, blockIdx.x * 16, parts, wave, DOWN_WAVES);
#pragma unroll
  for (int i = 0; i < H_CHUNKS; ++i) {
    const int c = tid + i * NT, row = c / per_row;
    if (c < chunks) *(u32x4_a*)(h_lds + row * h_row + (c - row * per_row) * 8) = hv[i];
  }
  if (tid < pairs) {
    prob[tid] = pair_weight(a, picked + tid / a.k * a.k, tid % a.k);
    if (blockIdx.x == 0) a.probs[tid] = prob[tid];
  }
  __syncthreads();
  d.run([&](int which, int part, int, const f32x4& sum) {
    if (d.r < s.item_count[which]) *(f32x4*)(partial + (((s.item_first[which] + d.r) * parts + part) * 16 + d.g * 4)) = sum;
  });
  __syncthreads();
  for (int i = tid; i < a.T * 16; i += NT) {
    const int t = i >> 4, c = i & 15;
    float sum = 0.f;
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
      const float p = prob[t * a.k + j];
      const float* v = partial + spot[t * a.k + j] * parts * 16 + c;
      float y = 0.f;
      for (int q = 0; q < parts; ++q) y += v[q * 16];
      if (p != 0.f) sum = fmaf(p, y, sum);           // (a weight of 0 adds nothing, not even 0 * infinity)
    }
    ((X*)a.out)[(int64_t)t * a.out_stride + blockIdx.x * 16 + c] = (X)sum;
  }
}

// More of them: grid (H / 64, z), a block makes 64 columns of the pairs of its share of the items, which go to memory as
// y[part][pair][H] in 32 bits; combine_kernel adds them up.  Four tiles beside each other use a load of h four times: with one
// (and all items in one block, no memory between) the loads' addresses took longer than the weights: 64 tokens, 8 of 128 experts
// of 1024 x 4096 155 us, so 106 and 5 for the sum; 11 tokens, 2 of 8 of 4096 x 2048 in bf16 50, so 29 and 5.
template <class W, int PER>
__device__ void down_many_kernel(const MoeArgs& a) {
  __shared__ SortLds s;
  constexpr int NT = DOWN_MANY_WAVES * 64;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), pairs = a.T * a.k;
  int expert[MOE_T * MOE_K / NT];
#pragma unroll
  for (int i = 0; i < MOE_T * MOE_K / NT; ++i) expert[i] = tid + i * NT < pairs ? a.ids[tid + i * NT] : 0;
  sort_pairs<NT, PER>(a, s, expert, [](int, int) {});
  const int waves = gridDim.y * DOWN_MANY_WAVES;
  const int parts = max(1, min(waves / s.items, a.max_parts));
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *a.parts = parts;
  const int n0 = blockIdx.x * DOWN_MANY_COLS;
  DownWave<W, DOWN_MANY_COLS / 16, 2, false, PER> d(a, s, nullptr, n0, parts, wave * gridDim.y + blockIdx.y, waves);
  d.run([&](int which, int part, int t, const f32x4& sum) {
    if (d.r < s.item_count[which] && n0 + t * 16 < a.H)
      *(f32x4*)(a.y + ((int64_t)part * pairs + s.pair[s.item_first[which] + d.r]) * a.H + n0 + t * 16 + d.g * 4) = sum;
  });
}

// out[t, c] = sum over places of their weight times the sum over parts; grid (H / 1024, T), four columns a thread
template <class X>
__device__ void combine_kernel(const MoeArgs& a) {
  __shared__ float weight[MOE_K];
  const int tid = threadIdx.x, t = blockIdx.y, c = (blockIdx.x * 256 + tid) * 4;
  const int parts = *a.parts;
  const int64_t plane = (int64_t)a.T * a.k * a.H;
  const float* v = a.y + (int64_t)t * a.k * a.H + min(c, a.H - 4);
  // (the first parts of the first places are on their way before the weights are there)
  constexpr int AHEAD = 8;
  f32x4 ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) ahead[j] = *(const f32x4*)(v + (int64_t)min(j, a.k - 1) * a.H);
  if (tid < a.k) {
    weight[tid] = pair_weight(a, a.picked + t * a.k, tid);
    if (blockIdx.x == 0) a.probs[t * a.k + tid] = weight[tid];
  }
  __syncthreads();
  if (c >= a.H) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int j, f32x4 y) {
#pragma unroll 4
    for (int q = 1; q < parts; ++q) y += *(const f32x4*)(v + (int64_t)j * a.H + q * plane);
    const float p = weight[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = p != 0.f ? fmaf(p, y[i], sum[i]) : sum[i];      // (a weight of 0 adds nothing, not even 0 * infinity)
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (j < a.k) add(j, ahead[j]);
  for (int j = AHEAD; j < a.k; ++j) add(j, *(const f32x4*)(v + (int64_t)j * a.H));
  X* o = (X*)a.out + (int64_t)t * a.out_stride + c;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (X)sum[i];
}

}  // namespace kcg_ops
