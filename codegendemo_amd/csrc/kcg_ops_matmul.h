// kcg_ops_matmul.h — product of e4m3 operands with a scale for each 128 values of a row of A and each 128 x 128 block of B:
//   C[m, n] = sum_g sa[m, g] sb[n / 128, g] sum_{k in group g} A[m, k] B[n, k]
// A 16 x 16 x 128 product (E4m3Dot, or WideDot for float32 results) covers exactly one group of k, so its result is the
// inner sum; it is scaled and added to the float32 accumulator by one fma per element.  B is the first matrix operand: a lane then holds 4 consecutive n of ONE m,
// needs one activation scale, and stores 4 neighbours of a row of C.
#pragma once
#include "kcg_ops_common.h"

namespace kcg_ops {

// ---------------------------------------------------------------------------------------------
// Few rows (M <= 16 CT): bound by the bytes of B and, from some 16 rows on, by what its blocks read of A between them.  A
// block owns 16 RT rows of B; its NW waves split K, every byte of B goes from memory straight into the matrix operand (an
// instruction reads 64 bytes of 16 rows, the next one the rest of those lines), and the partial sums meet in LDS, added
// in wave order (the same result on every run).  RT = 2 halves the reads of A for each byte of B.
// ---------------------------------------------------------------------------------------------
template <class TC, int CT, int RT, int NW>
__device__ void skinny_kernel(const MatmulArgs& p, f32x4* red) {
  typedef typename DotOf<TC>::type Dot;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * RT;
  const uint8_t* b[RT];
#pragma unroll
  for (int q = 0; q < RT; ++q) b[q] = p.b + (int64_t)min(n0 + q * 16 + r, p.N - 1) * p.ldb;   // (rows beyond N: computed from one that exists, not stored)
  const float* sb = p.sb + (int64_t)(n0 / GROUP) * p.sb_n;       // (16 RT rows from a multiple of 16 RT lie in one block of 128)
  const uint8_t* a[CT];
  const float* sa[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int64_t m = min(t * 16 + r, p.M - 1);
    a[t] = p.a + m * p.lda;
    sa[t] = p.sa + m * p.sa_m;
  }
  f32x4 acc[RT][CT];
#pragma unroll
  for (int q = 0; q < RT; ++q)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // U groups from kb on, all their loads in front of the first product
  auto groups = [&](auto u_c, auto whole_c, int kb) {
    constexpr int U = decltype(u_c)::value;
    constexpr bool WHOLE = decltype(whole_c)::value;
    i32x8 bq[U][RT], aq[U][CT];
    float s[U][CT], sbv[U];
    auto load = [&](const uint8_t* row, int k) {
      if constexpr (WHOLE) return join(*(const u32x4_a*)(row + k), *(const u32x4_a*)(row + k + 64));
      else return join(load16_masked(row, k, p.K), load16_masked(row, k + 64, p.K));
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < RT; ++q) bq[u][q] = load(b[q], (kb + u) * GROUP + g * 16);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        aq[u][t] = load(a[t], (kb + u) * GROUP + g * 16);
        s[u][t] = sa[t][(kb + u) * p.sa_k];
      }
      sbv[u] = sb[(kb + u) * p.sb_k];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      typename Dot::frag bf[RT];
#pragma unroll
      for (int q = 0; q < RT; ++q) bf[q] = Dot::make(bq[u][q]);
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const typename Dot::frag af = Dot::make(aq[u][t]);
        const float f = s[u][t] * sbv[u];
#pragma unroll
        for (int q = 0; q < RT; ++q) {
          const f32x4 d = Dot::mma(bf[q], af);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[q][t][i] = fmaf(d[i], f, acc[q][t][i]);
        }
      }
    }
  };
  constexpr int U = CT == 1 ? 4 : 2;
  int kb = p.KB * wave / NW;
  const int to = p.KB * (wave + 1) / NW, whole = min(to, p.K / GROUP);
  for (; kb + U <= whole; kb += U) groups(Int<U>(), Int<1>(), kb);
  for (; kb < to; ++kb) groups(Int<1>(), Int<0>(), kb);            // the rest, the partial last group among it
  constexpr int TILES = RT * CT;
#pragma unroll
  for (int q = 0; q < RT; ++q)
#pragma unroll
    for (int t = 0; t < CT; ++t) red[(wave * TILES + q * CT + t) * 64 + lane] = acc[q][t];
  __syncthreads();
  for (int i = threadIdx.x; i < TILES * 64; i += NW * 64) {
    f32x4 v = red[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += red[w * TILES * 64 + i];
    const int tile = i >> 6, q = tile / CT, t = tile - q * CT;
    const int m = t * 16 + (i & 15), n = n0 + q * 16 + ((i >> 4) & 3) * 4;
    if (m < p.M && n < p.N) store4((TC*)p.c + (int64_t)m * p.ldc + n, v, p.N - n, p.c_wide);
  }
}

// ---------------------------------------------------------------------------------------------
// Tiles of BM x BN, WM x WN waves, K in steps of one group (128 bytes of a row).
// LDS: S stages of BM + BN rows of 128 bytes, filled by global_load_lds (16 bytes a lane, no registers).  The chunk at
// place c of row r is chunk c ^ (r & 7) of that row: 8 lanes that read one chunk column of 8 rows touch all banks.
// A wave keeps its activation fragments (MB x 16 columns) for a K step and streams the weight fragments (NB x 16 rows)
// past them, two ahead.  A step ends (barrier, fetch into the stage it has read) in front of the last weight row, whose
// fragments are in registers by then: with S = 2 a fetch has most of a step to land, with more stages S - 1 steps; the
// fragment reads of the next step run under the last row's matrix instructions, and the fma of a product under the next
// two products.
// KS > 1: KS groups of WM x WN waves take the steps in turn, each with stages of its own, and their sums meet in LDS.  A step
// of a small tile is a chain of waits (0.28 us, whatever the number of tiles): this shortens the chain where tiles are few.
// Scales come the same way in chunks of 8 steps, a chunk ahead: read per lane and step where they are needed, from rows
// of their own, they made 4096^3 take 88 us, with rows side by side 70.
// ---------------------------------------------------------------------------------------------
template <int BM, int BN, int WM, int WN, int S, int KS>
struct TilePlan {
  static constexpr int NT = WM * WN * 64;          // threads of a group
  static constexpr int MB = BM / WM / 16, NB = BN / WN / 16;
  static constexpr int ROWS = BM + BN, STAGE = ROWS * GROUP;
  static constexpr int FETCH = ROWS * 8 / NT;      // 16-byte chunks a thread fetches for a stage
  static constexpr int RPF = NT / 8;               // rows one fetch of all threads covers
  // Pieces of a fetch: LAST behind the barrier, the others over the first rows of the next step where the tile is large (all
  // at once, its waves stand in front of the one address unit, 16 cycles an instruction, and the matrix cores behind them:
  // 8192^3 488 us, so 478); small tiles wait for memory, not for the unit (2048^3 19.7 us, all at once 17.3).
  static constexpr int LAST = NB > 4 ? 2 : FETCH;
  static constexpr int PER_ROW = (FETCH - LAST + NB / 2 - 1) / (NB / 2);
  static constexpr int SB = BN >= GROUP ? BN / GROUP : 1;              // blocks of 128 rows of B a tile has scales from
  static constexpr int STEPS = 8;                                      // of a chunk of scales
  static constexpr int SCALES = STEPS * BM + 64;                       // floats of one: [step][row], then [block][step]
  static constexpr int PART = S * STAGE + 2 * SCALES * 4, LDS = KS * PART;
  static_assert((KS - 1) * BM * BN * 4 <= LDS, "the groups' sums");
  static_assert(BM % RPF == 0 && BN % RPF == 0 && NB >= 2 && NB % 2 == 0 && (S & (S - 1)) == 0 && SB * STEPS <= 64, "tile plan");
  static_assert(BN / WN <= GROUP && GROUP % (BN / WN) == 0, "a wave's rows of B lie in one block of 128");
  static_assert(S == 2 || LAST == FETCH, "the waits count whole fetches");
  static_assert((BM % 64 == 0 || 64 % BM == 0) && STEPS * BM / 64 % (NT / 64) == 0, "scales: whole waves");
};

// 16 (4) bytes a lane from base + off into consecutive LDS from lds on.  In assembly, because the compiler would wait for every
// such fetch in front of each later LDS read; the waits that are needed are written out in the kernel.  (No output
// registers; vmcnt counts it, which makes the compiler's own waits stricter, never weaker.)
__device__ __forceinline__ void fetch_lds16(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void fetch_lds4(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

template <class TC, int BM, int BN, int WM, int WN, int S, int KS>
__device__ void tile_kernel(const MatmulArgs& p, uint8_t* lds) {
  typedef TilePlan<BM, BN, WM, WN, S, KS> P;
  typedef typename DotOf<TC>::type Dot;
  constexpr int MB = P::MB, NB = P::NB, NW = WM * WN;
  const int lane = threadIdx.x & 63, wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = KS > 1 ? wave_id / NW : 0, wave = wave_id - kg * NW, tid = wave * 64 + lane;     // group, and place in it
  const int wm = wave % WM, wn = wave / WM;
  const int r = lane & 15, g = lane >> 4;
  uint8_t* const smem = lds + kg * P::PART;

  // block -> tile: ids are dealt round-robin to the 8 XCDs; each gets one contiguous part of the order, which walks the
  // n tiles of 4 tile rows together, so that an XCD's resident tiles share panels of both operands in its L2
  int bid = blockIdx.x;
  const int total = p.grid_m * p.grid_n;
  {
    const int per = total >> 3, left = total & 7, xcd = bid & 7;
    bid = xcd * per + min(xcd, left) + (bid >> 3);
  }
  constexpr int GM = 4;
  const int gsize = GM * p.grid_n, grp = bid / gsize, in = bid - grp * gsize;
  const int gm = min(GM, p.grid_m - grp * GM);
  const int tm = grp * GM + in % gm, tn = in / gm;
  const int m0 = tm * BM, n0 = tn * BN;
  // step t of this group is group kb(t) of K; it has `steps` of them, every group at least p.KB / KS
  const int steps = (p.KB - kg + KS - 1) / KS, last_step = (p.KB - 1) / KS;
  auto group_of = [&](int t) { return t * KS + kg; };

  // fetch: thread -> row tid / 8 (+ RPF per further piece), place tid % 8
  const int frow = tid >> 3, fchunk = (tid & 7) ^ (frow & 7);     // (RPF is a multiple of 8: the swizzle is the same in every piece)
  const uint8_t* abase = p.a + (int64_t)m0 * p.lda;
  const uint8_t* bbase = p.b + (int64_t)n0 * p.ldb;
  constexpr int FA = BM / P::RPF, FB = BN / P::RPF;
  unsigned off[FA + FB];
#pragma unroll
  for (int f = 0; f < FA; ++f) off[f] = (unsigned)(min(frow + f * P::RPF, p.M - 1 - m0) * (unsigned)p.lda) + fchunk * 16;
#pragma unroll
  for (int f = 0; f < FB; ++f) off[FA + f] = (unsigned)(min(frow + f * P::RPF, p.N - 1 - n0) * (unsigned)p.ldb) + fchunk * 16;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const unsigned lds_wave = lds0 + wave * 1024;
  // a chunk of the partial last group that lies behind K: the row's first chunk of that group instead (cleared in LDS later)
  const bool ragged = (p.K & (GROUP - 1)) != 0;
  const bool behind = ragged && fchunk * 16 >= (p.K & (GROUP - 1));
  auto fetch = [&](auto from_c, auto to_c, int t) {        // pieces [from, to) of FETCH
    const int kb = group_of(t);
    const unsigned back = behind && kb == p.KB - 1 ? fchunk * 16 : 0;
    const unsigned to = lds_wave + (t & (S - 1)) * P::STAGE;
    const uint8_t* ak = abase + (int64_t)kb * GROUP;
    const uint8_t* bk = bbase + (int64_t)kb * GROUP;
    static_for<decltype(from_c)::value, decltype(to_c)::value>([&](auto f_c) {
      constexpr int f = decltype(f_c)::value;
      fetch_lds16(f < FA ? ak : bk, off[f] - back, to + f * P::RPF * GROUP);
    });
  };
  // zeros behind K in the stage of the partial last group
  auto clear_tail = [&](int t) {
    if (group_of(t) != p.KB - 1) return;
    const int kt = p.K & (GROUP - 1);
    uint8_t* st = smem + (t & (S - 1)) * P::STAGE;
    for (int i = tid; i < P::ROWS * 8; i += P::NT) {
      const int row = i >> 3, c = i & 7;
      u32x4_a* at = (u32x4_a*)(st + row * GROUP + ((c ^ (row & 7)) << 4));
      const int n = kt - c * 16;
      if (n < 16) {
        u32x4 v = *at;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = n - 4 * w;
          v[w] = left >= 4 ? v[w] : left <= 0 ? 0u : v[w] & (0xffffffffu >> (32 - 8 * left));
        }
        *at = v;
      }
    }
  };
  // lane's two chunks of a row: g and g + 4 (as good a split of the 128 k values as any, and free of bank conflicts)
  const unsigned sw0 = ((g ^ (r & 7)) << 4), sw1 = (((g + 4) ^ (r & 7)) << 4);
  const uint8_t* arow = smem + (wm * MB * 16 + r) * GROUP;
  const uint8_t* brow = smem + (BM + wn * NB * 16 + r) * GROUP;
  auto frag = [&](const uint8_t* base, int i, int t) {
    const uint8_t* q = base + (t & (S - 1)) * P::STAGE + i * 16 * GROUP;
    return join(*(const u32x4_a*)(q + sw0), *(const u32x4_a*)(q + sw1));
  };
  // scales of chunk c (the group's steps 8 c .. 8 c + 7): an instruction fetches 64 rows of one step, the last one those of the weights
  constexpr int STEPS = P::STEPS;
  const float* const scales = (const float*)(smem + S * P::STAGE);
  const unsigned sa_step = (unsigned)p.sa_k * KS, sb_step = (unsigned)p.sb_k * KS;
  auto fetch_scales = [&](int c) {
    const unsigned to = lds0 + S * P::STAGE + (c & 1) * P::SCALES * 4;
    const int most = steps - 1 - c * STEPS;
    const float* base = p.sa + (int64_t)m0 * p.sa_m + (int64_t)group_of(c * STEPS) * p.sa_k;
#pragma unroll
    for (int i = 0; i < STEPS * BM / 64 / NW; ++i) {
      const int at = (wave + i * NW) * 64 + lane, step = min(at / BM, most), row = min(at % BM, p.M - 1 - m0);
      fetch_lds4(base, ((unsigned)row * (unsigned)p.sa_m + (unsigned)step * sa_step) * 4u, to + (wave + i * NW) * 256);
    }
    if (wave == 0) {
      const float* sb = p.sb + (int64_t)(n0 / GROUP) * p.sb_n + (int64_t)group_of(c * STEPS) * p.sb_k;
      const int block = min(min(lane / STEPS, P::SB - 1), (p.N - 1) / GROUP - n0 / GROUP), step = min(lane % STEPS, most);
      fetch_lds4(sb, ((unsigned)block * (unsigned)p.sb_n + (unsigned)step * sb_step) * 4u, to + STEPS * BM * 4);
    }
  };
  const float* my_sa = scales + wm * MB * 16 + r;
  const float* my_sb = scales + STEPS * BM + (n0 % GROUP + wn * NB * 16) / GROUP * STEPS;
  float s[MB], s_next[MB], sb_next;
  auto read_scales = [&](float (&v)[MB], int t) {
    const int chunk = ((t / STEPS) & 1) * P::SCALES, step = t % STEPS;
#pragma unroll
    for (int j = 0; j < MB; ++j) v[j] = my_sa[chunk + step * BM + j * 16];
    sb_next = my_sb[chunk + step];
  };

  f32x4 acc[NB][MB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (p.KB > 0) {
    if (steps > 0) {
      fetch_scales(0);
      static_for<0, S - 1>([&](auto t_c) {
        constexpr int t = decltype(t_c)::value;
        if (t < steps) fetch(Int<0>(), Int<P::FETCH>(), t);
      });
    }
    // (in order: the first stage and the scales in front of it have landed when no more than the other stages are left)
    if (steps >= S - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * P::FETCH) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (ragged && last_step == 0) {
      clear_tail(0);
      __syncthreads();
    }
    if (S - 1 < steps) fetch(Int<0>(), Int<P::LAST>(), S - 1);
    i32x8 am[MB], bn[4];                         // weight row i in place i % 4, two rows ahead of its products
    // (a group without a step reads what lies there, and uses none of it)
    read_scales(s, 0);
#pragma unroll
    for (int j = 0; j < MB; ++j) s[j] *= sb_next;
#pragma unroll
    for (int j = 0; j < MB; ++j) am[j] = frag(arow, j, 0);
    bn[0] = frag(brow, 0, 0);
    bn[1] = frag(brow, 1, 0);
    // Products q = i MB + j run through d[q % 3]; the fma of a product follows the second product behind it, when its result is
    // there without a wait.
    f32x4 d[3];
    auto add = [&](auto q_c) {
      constexpr int q = decltype(q_c)::value, i = q / MB, j = q % MB;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[q % 3][e], s[j], acc[i][j][e]);
      // (here, not behind the branches at the end of the step, where the compiler would gather them and keep every d until then)
      asm volatile("" : "+v"(acc[i][j]));
    };
    auto step = [&](int t) {
      const int nx = min(t + 1, steps - 1);
      typename Dot::frag af[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) af[j] = Dot::make(am[j]);
      // (behind the stages fetched so far, in front of the ones to come: the waits below cover them)
      if (t % STEPS == 1 && t - 1 + STEPS < steps) fetch_scales(t / STEPS + 1);
      static_for<0, NB>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        if constexpr (i == NB - 1) {
          // every fragment of this stage is in registers or on its way; the next stage has landed when no more than the S - 2
          // behind it are left
          if (S > 2 && t + S - 1 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * P::FETCH) : "memory");
          else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          read_scales(s_next, nx);
          if (ragged && t + 1 == last_step) {
            clear_tail(t + 1);
            __syncthreads();
          }
          if (t + S < steps) fetch(Int<0>(), Int<P::LAST>(), t + S);
        } else if constexpr (P::LAST + i * P::PER_ROW < P::FETCH) {
          constexpr int to = P::LAST + (i + 1) * P::PER_ROW;
          if (t + S - 1 < steps) fetch(Int<P::LAST + i * P::PER_ROW>(), Int<(to < P::FETCH ? to : P::FETCH)>(), t + S - 1);
        }
        if constexpr (i + 2 < NB) bn[(i + 2) % 4] = frag(brow, i + 2, t);
        const typename Dot::frag bf = Dot::make(bn[i % 4]);
        static_for<0, MB>([&](auto j_c) {
          constexpr int j = decltype(j_c)::value, q = i * MB + j;
          d[q % 3] = Dot::mma(bf, af[j]);
          if constexpr (i == NB - 1) am[j] = frag(arow, j, nx);          // (after the last step: the same stage again, unused)
          if constexpr (i == NB - 1 && j == 0) bn[0] = frag(brow, 0, nx);
          if constexpr (i == NB - 1 && j == (NB > 2 && MB > 1 ? 1 : MB - 1)) bn[1] = frag(brow, 1, nx);   // (NB = 2: row 1 is this row)
          if constexpr (q >= 2) add(Int<q - 2>());
          __builtin_amdgcn_sched_barrier(0);
        });
      });
      add(Int<NB * MB - 2>());
      add(Int<NB * MB - 1>());
#pragma unroll
      for (int j = 0; j < MB; ++j) s[j] = s_next[j] * sb_next;
    };
    // the steps that every group has, then those that only some have: the others keep them company at the barrier
    const int common = p.KB / KS;
    for (int t = 0; t < common; ++t) step(t);
    if constexpr (KS > 1) {
      if (common * KS < p.KB) {
        if (common < steps) step(common);
        else __builtin_amdgcn_s_barrier();
      }
      // sums of groups 1 .. KS - 1, in LDS behind the last reads of it, added by group 0 in their order
      __syncthreads();
      f32x4* sums = (f32x4*)lds;
      if (kg > 0) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int j = 0; j < MB; ++j) sums[(((kg - 1) * NW + wave) * NB * MB + i * MB + j) * 64 + lane] = acc[i][j];
      }
      __syncthreads();
      if (kg > 0) return;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
          for (int o = 0; o < KS - 1; ++o) acc[i][j] += sums[((o * NW + wave) * NB * MB + i * MB + j) * 64 + lane];
    }
  }
  if constexpr (KS == 1) {
    // A lane's four results are 8 (16) bytes of a row and 16 rows lie under an instruction: stored like that, a line comes to L2
    // in pieces.  So a wave lays its part of the tile out in LDS first (chunk c of row m in place c ^ m: no two rows of a write in
    // one bank) and stores whole rows of it, 16 bytes a lane.  (bf16, 4096 x 4096 x 512: 19.1 us from the registers, 16.0 so; by
    // tiles of 128 x 128, K = 1024: 28.9, 24.4.)
    constexpr int EPC = 16 / sizeof(TC), CH = NB * 16 / EPC, RPI = 64 / CH;       // elements of a chunk, chunks of a row, rows an instruction
    static_assert(P::NT / 64 * MB * 16 * CH * 16 <= P::LDS && CH <= 64 && (CH & (CH - 1)) == 0, "the tile in LDS");
    __syncthreads();                               // (every wave has read its last fragments)
    uint8_t* const part = lds + wave * (MB * 16 * CH * 16);
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        TC t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = (TC)acc[i][j][e];
        const int m = j * 16 + r, at = (i * 16 + g * 4) * (int)sizeof(TC);
        uint8_t* q = part + (m * CH + ((at >> 4) ^ (m & (CH - 1)))) * 16 + (at & 15);
        if constexpr (sizeof(TC) == 4) *(u32x4_a*)q = *(u32x4_a*)t;
        else *(u32x2_a*)q = *(u32x2_a*)t;
      }
    const int chunk = lane % CH, n = n0 + wn * NB * 16 + chunk * EPC;
#pragma unroll
    for (int i = 0; i < MB * 16 / RPI; ++i) {
      const int row = i * RPI + lane / CH, m = m0 + wm * MB * 16 + row;
      const u32x4 v = *(const u32x4_a*)(part + (row * CH + (chunk ^ (row & (CH - 1)))) * 16);
      if (m < p.M && n < p.N) {
        TC* c = (TC*)p.c + (int64_t)m * p.ldc + n;
        if (n + EPC <= p.N) {
          *(u32x4_u*)c = v;
        } else {
          TC t[EPC];
          *(u32x4_a*)t = v;
#pragma unroll
          for (int e = 0; e < EPC; ++e)
            if (n + e < p.N) c[e] = t[e];
        }
      }
    }
  } else {
    if (kg > 0) return;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int m = m0 + (wm * MB + j) * 16 + r;
      if (m < p.M) {
        TC* c = (TC*)p.c + (int64_t)m * p.ldc;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int n = n0 + wn * NB * 16 + i * 16 + g * 4;
          if (n < p.N) store4(c + n, acc[i][j], p.N - n, p.c_wide);
        }
      }
    }
  }
}

}  // namespace kcg_ops
