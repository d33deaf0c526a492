// kcg_ops.cc — host side of the operators declared in include/kcg_ops.h: argument checks, the choice of a kernel, launches.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <string>

#include "../../include/kcg_gemm.h"
#include "../../include/kcg_ops.h"
#include "kcg_host.h"
#include "kcg_ops_args.h"

// the code object of kcg_ops.hip; empty in a library that was built where there is no hipcc
#ifdef KCG_OPS_CODE
__asm__(".section .rodata\n.balign 4096\n.global kcg_ops_code\nkcg_ops_code:\n.incbin \"" KCG_OPS_CODE "\"\n.byte 0\n.previous\n");
extern "C" const char kcg_ops_code[];
#else
static const char kcg_ops_code[] = "";
#endif

namespace {

using kcg::host_fail;
using kcg::host_hip;
using kcg::host_hip_fail;
using kcg::HostHip;
using namespace kcg_ops;

// ---- kernels ---------------------------------------------------------------------------------
// The tiles of the 8-bit product (kcg_ops_matmul.h).  A call takes the one that this estimate of its time, in microseconds,
// is smallest for: every round of blocks costs start + steps * step, where a round is one block on each of the 256 compute
// units, or two where two fit one (step2: their step); steps = groups of 128 of K / ks.  Products with float32 results take
// nearly twice the matrix instructions a step, so they have costs of their own.  Measured at N, K in {1024 .. 16384}; the
// estimates lie within 10 % of what was measured, some 20 % at the largest sizes and between one round and two.  The figures beside
// the tiles, and at the other choices below, are microseconds a call in a graph of calls, both sides on one card.
struct Cost {
  float start, step, step2;
};
struct Tile {
  const char* name;
  int bm, bn, ks, threads;
  Cost half, full;                                        // 16-bit results, float32 results
};
const Tile kTileTable[] = {
    {"32x32_2x1x4", 32, 32, 4, 512, {1.6f, .39f, 0.f}, {1.9f, .64f, 0.f}},        // 37 x 4096 x 4096: 7.9 us (64 x 64: 12.9)
    {"64x32_4x1x2", 64, 32, 2, 512, {1.2f, .36f, 0.f}, {1.4f, .62f, 0.f}},        // 37 x 8192 x 4096: 10.1 (32 x 32: 13.4, 64 x 64 by two: 11.3)
    {"64x64_2x2x1", 64, 64, 1, 256, {.4f, .305f, .52f}, {1.2f, .52f, .74f}},      // 512 x 4096 x 1024: 7.8 (by two: 11.2)
    {"64x64_2x2x2", 64, 64, 2, 512, {1.9f, .47f, 0.f}, {2.2f, .76f, 0.f}},        // 256 x 4096 x 4096: 12.2 (by one: 13.4)
    {"64x128_2x2x1", 64, 128, 1, 256, {.8f, .6f, .67f}, {1.6f, .74f, 1.07f}},     // 4096 x 1536 x 1000, float32: 22.7 (64 x 64: 28.3, 128 x 128: 24.1)
    {"128x128_2x2x1", 128, 128, 1, 256, {1.6f, .655f, 1.1f}, {4.6f, 1.08f, 1.75f}},  // 2048 x 4096 x 4096: 40.5 (8 waves: 46.9)
    // for 16-bit results only: the next two are no faster than 64 x 64 and 64 x 128 with float32 ones, the last has no registers for them
    {"128x64_4x2x1", 128, 64, 1, 512, {.6f, .5f, 0.f}, {}},                       // 128 x 16384 x 4096: 17.8 (64 x 64: 18.5)
    {"128x128_4x2x1", 128, 128, 1, 512, {2.f, .575f, 0.f}, {}},                   // 1024 x 4096 x 4096: 24.3 (4 waves: 27.4)
    {"256x256_4x2x1", 256, 256, 1, 512, {7.f, 1.55f, 0.f}, {}},                   // 4096^3: 64.7 (128 x 128: 91.3)
};
constexpr int kTiles = sizeof(kTileTable) / sizeof(kTileTable[0]), kTilesF32 = kTiles - 3;
constexpr double kLaunch = 2.3;

double tile_estimate(const Tile& v, const Cost& c, int64_t m, int64_t n, int64_t groups) {
  const double tiles = (double)((m + v.bm - 1) / v.bm) * (double)((n + v.bn - 1) / v.bn), steps = (double)((groups + v.ks - 1) / v.ks);
  if (c.step2 == 0.f) return kLaunch + std::ceil(tiles / 256) * (c.start + steps * c.step);
  const double full = std::floor(tiles / 512), rest = tiles - 512 * full;
  return kLaunch + full * (c.start + steps * c.step2) + (rest > 0 ? c.start + steps * (rest <= 256 ? c.step : c.step2) : 0);
}
// 17 to 32 rows without a tile (rt: 16-row tiles of b a block): N / 16 / rt blocks
double skinny_estimate(int rt, int64_t n, int64_t groups) {
  const double rounds = (double)((n + 16 * rt - 1) / (16 * rt)) / 256;
  return 2.2 + groups * (rt == 1 ? .172 : .24) * (rounds > 1 ? rounds : 1);
}

enum { kNorm = 0, kSwiglu = kNorm + 21, kSkinny = kSwiglu + 3, kTile = kSkinny + 12, kMoeUp = kTile + 3 * kTiles, kMoeFew = kMoeUp + 3, kMoeMany = kMoeFew + 3, kMoeCombine = kMoeMany + 4, kNumKernels = kMoeCombine + 2 };

std::string kernel_symbol(int i) {
  static const char* const types[3] = {"bf16", "f16", "f32"};
  static const char* const norm[7] = {"64_1", "128_1", "256_1", "512_1", "1024_1", "1024_2", "1024_0"};
  static const char* const moe[3] = {"e4m3_bf16", "e4m3_f16", "bf16_bf16"};
  if (i < kSwiglu) return std::string("kcg_norm_") + types[i / 7] + "_" + norm[i % 7];
  if (i < kSkinny) return std::string("kcg_swiglu_") + types[i - kSwiglu];
  if (i < kTile) {
    const int v = (i - kSkinny) % 4;
    return std::string("kcg_mm8_skinny_") + types[(i - kSkinny) / 4] + "_" + std::to_string(v / 2 + 1) + "x" + std::to_string(v % 2 + 1);
  }
  if (i < kMoeUp) return std::string("kcg_mm8_tile_") + types[(i - kTile) / kTiles] + "_" + kTileTable[(i - kTile) % kTiles].name;
  if (i < kMoeFew) return std::string("kcg_moe_up_") + moe[i - kMoeUp];
  if (i < kMoeMany) return std::string("kcg_moe_down_few_") + moe[i - kMoeFew];
  if (i < kMoeCombine) return std::string("kcg_moe_down_many_") + ((i - kMoeMany) / 2 ? "bf16_" : "e4m3_") + ((i - kMoeMany) % 2 ? "16" : "8");
  return i == kMoeCombine ? "kcg_moe_combine_bf16" : "kcg_moe_combine_f16";
}

// What a product of these sizes (m, n > 0) with results of type t (0: bf16, 1: f16, 2: f32) runs.
struct MatmulChoice {
  int fn, threads, grid_m, grid_n;
  int64_t blocks;
};
MatmulChoice choose_matmul(int64_t m, int64_t n, int64_t k, int t) {
  const int64_t groups = (k + 127) / 128;
  int rt = 0, tile = 0;                    // rt > 0: without a tile
  if (m <= 16) {
    rt = n >= 32 * 224 ? 2 : 1;            // 32 rows of b a block where that still fills the chip (8 x 8192 x 4096: 8.6, with 16 rows 9.9)
  } else {
    double best = 1e30;
    for (int v = 0; v < (t == 2 ? kTilesF32 : kTiles); ++v) {
      const double e = tile_estimate(kTileTable[v], t == 2 ? kTileTable[v].full : kTileTable[v].half, m, n, groups);
      if (e < best) {
        best = e;
        tile = v;
      }
    }
    if (m <= 32)
      for (int r = 1; r <= 2; ++r) {
        const double e = skinny_estimate(r, n, groups);
        if (e < best) {
          best = e;
          rt = r;
        }
      }
  }
  if (rt) return {kSkinny + t * 4 + (int)(m - 1) / 16 * 2 + rt - 1, SKINNY_WAVES * 64, 0, 0, (n + 16 * rt - 1) / (16 * rt)};
  const Tile& v = kTileTable[tile];
  const int64_t gm = (m + v.bm - 1) / v.bm, gn = (n + v.bn - 1) / v.bn;
  return {kTile + t * kTiles + tile, v.threads, (int)gm, (int)gn, gm * gn};
}

struct DeviceKernels {
  hipModule_t module;
  hipFunction_t fn[kNumKernels];
};

// `device` current while it lives, the caller's device again afterwards
struct OnDevice {
  const HostHip* hip;
  int before = -1;
  hipError_t error;
  OnDevice(const HostHip* h, int device) : hip(h) {
    int now = -1;
    error = hip->GetDevice(&now);
    if (error == hipSuccess && now != device) {
      error = hip->SetDevice(device);
      if (error == hipSuccess) before = now;
    }
  }
  ~OnDevice() {
    if (before >= 0) (void)hip->SetDevice(before);
  }
};

// LDS of a block of the experts' second kernel for few tokens: 16 partial sums for each pair and part of I, of which there are
// tokens * 16 at most (parts = 16 / items, and items >= topk <= 16), and h beside them.
int moe_partial_bytes(int64_t tokens) { return (int)(tokens * 16 * 16 * 4); }
int64_t moe_h_bytes(int64_t pairs, int64_t inter) { return 2 * pairs * (inter + 8) * 2; }

int64_t groups(int64_t n) { return (n + 127) / 128; }

// How a call's workspace is laid out and its second product shared out.
struct MoePlan {
  int64_t slots, plane, parts_at, y_at, bytes;     // bytes of one plane of h; where the number of parts and y stand
  bool few;                                        // h fits LDS: one kernel for the second product and the sum
  int per, z, max_parts;                           // pairs an item holds, blocks that share the items, most parts of I
};
MoePlan moe_plan(int64_t tokens, int64_t experts, int64_t topk, int64_t hidden, int64_t inter) {
  MoePlan m = {};
  const int64_t pairs = tokens * topk, cols = (hidden + DOWN_MANY_COLS - 1) / DOWN_MANY_COLS;
  m.slots = pairs < experts ? pairs : experts;
  m.plane = pairs * inter * 2;
  // 16 columns of out a block: with fewer blocks than compute units only the smallest calls gain (2 tokens, 8 of 128 experts of
  // 1024 x 4096: the call takes 48.2, the other way 52.9; 3 tokens, 2 of 8 of 4096 x 2048 in bf16, half as many blocks: 59.5, 59.4)
  m.few = tokens <= MOE_FEW && moe_h_bytes(pairs, inter) <= (hidden >= 16 * 256 ? MOE_H_LDS : MOE_H_LDS / 2);
  // one block on each of the 256 compute units; waves without an item of their own share I, in parts.  There are at least
  // `items` items: k experts, and `per` pairs an item.
  m.z = cols >= 256 ? 1 : (int)(256 / cols);
  // Items of 16 pairs halve the reads of W2 by experts of more than 8 tokens and cost the others four more loads a step: 64 tokens, 4 of 16
  // experts of 2048 x 4096: the call takes 126.7 (by eight 137.7), 2 of 8 of the same 73.9 (78.8); 8 tokens an expert (8 of 64 of 1024 x
  // 2048) cost nearly the same either way, 101.2 (103.7).
  m.per = pairs > 8 * experts ? 16 : 8;
  const int64_t items = std::max<int64_t>(std::max<int64_t>(topk, (pairs + m.per - 1) / m.per), 1);
  m.max_parts = (int)std::max<int64_t>(1, std::min<int64_t>(m.z * DOWN_MANY_WAVES / items, groups(inter)));
  m.parts_at = 2 * m.plane + pairs * 4;
  m.y_at = (m.parts_at + 4 + 15) / 16 * 16;
  m.bytes = tokens == 0 ? 0 : m.few ? m.y_at : m.y_at + m.max_parts * pairs * hidden * 4;
  return m;
}

// The kernels on `device` (current): loaded once per process and device, kept until the process ends.
int kernels_on(const HostHip* hip, int device, const DeviceKernels** out) {
  static std::mutex mu;
  static std::map<int, std::unique_ptr<DeviceKernels>> loaded;
  std::lock_guard<std::mutex> lock(mu);
  auto it = loaded.find(device);
  if (it == loaded.end()) {
    std::unique_ptr<DeviceKernels> k(new DeviceKernels);
    hipError_t e = hip->ModuleLoadData(&k->module, kcg_ops_code);
    if (e != hipSuccess) return host_hip_fail(e, "hipModuleLoadData (operators)");
    for (int i = 0; i < kNumKernels && e == hipSuccess; ++i) {
      if (i >= kTile + 2 * kTiles + kTilesF32 && i < kMoeUp) continue;       // tiles without a form for float32 results
      e = hip->ModuleGetFunction(&k->fn[i], k->module, kernel_symbol(i).c_str());
      // a block of the experts' second kernel for few tokens may use more than 64 KiB of LDS, part of it dynamic
      if (e == hipSuccess && i >= kMoeFew && i < kMoeMany)
        e = hip->FuncSetAttribute ? hip->FuncSetAttribute((const void*)k->fn[i], hipFuncAttributeMaxDynamicSharedMemorySize,
                                                          moe_partial_bytes(MOE_FEW) + MOE_H_LDS)
                                  : hipErrorNotSupported;
    }
    if (e != hipSuccess) {
      (void)hip->ModuleUnload(k->module);
      return host_hip_fail(e, "hipModuleGetFunction (operators)");
    }
    it = loaded.emplace(device, std::move(k)).first;
  }
  *out = it->second.get();
  return KCG_OK;
}

int launch(const HostHip* hip, hipFunction_t fn, unsigned gx, unsigned gy, unsigned block, unsigned lds, uint64_t stream, void* args) {
  void* params[1] = {args};
  const hipError_t e = hip->ModuleLaunchKernel(fn, gx, gy, 1, block, 1, 1, lds, (hipStream_t)(uintptr_t)stream, params, nullptr);
  return e == hipSuccess ? (int)KCG_OK : host_hip_fail(e, "hipModuleLaunchKernel");
}

// runs f(hip, kernels) with `device` current; nothing is thrown past it
template <class F>
int on_device(int device, F f) {
  try {
    if (!*kcg_ops_code) return host_fail(KCG_ERR_COMPILE, "the library was built without hipcc and has no kernels of the operators: build it again with hipcc");
    const HostHip* hip = host_hip();
    if (!hip) return KCG_ERR_HIP;
    OnDevice guard(hip, device);
    if (guard.error != hipSuccess) return host_hip_fail(guard.error, "hipSetDevice");
    const DeviceKernels* k = nullptr;
    if (int rc = kernels_on(hip, device, &k)) return rc;
    const int rc = f(hip, *k);
    if (rc == KCG_OK) kcg::host_clear_error();
    return rc;
  } catch (...) {
    return KCG_ERR_HIP;      // out of host memory while a message or a table was made
  }
}

int bad(const char* what) {
  try {
    return host_fail(KCG_ERR_ARGUMENT, what);
  } catch (...) {
    return KCG_ERR_ARGUMENT;
  }
}

// ---- checks ------------------------------------------------------------------------------------
int type_index(int64_t dtype) { return dtype == KCG_DT_BFLOAT16 ? 0 : dtype == KCG_DT_FLOAT16 ? 1 : dtype == KCG_DT_FLOAT32 ? 2 : -1; }
int type_bytes(int64_t dtype) { return dtype == KCG_DT_FLOAT32 ? 4 : dtype == KCG_DT_E4M3 ? 1 : 2; }
constexpr int64_t kMaxExtent = 1 << 30;       // rows and columns: 32-bit indices in the kernels, with room for a tile
constexpr int64_t kMaxStride = (int64_t)1 << 40;
constexpr int64_t kMaxThreads = UINT_MAX;     // of a launch
bool extent_ok(int64_t n) { return n >= 0 && n <= kMaxExtent; }
// a row stride: rows do not overlap (any value goes where there is one row)
bool stride_ok(int64_t stride, int64_t cols, int64_t rows) { return stride >= 0 && stride <= kMaxStride && (rows <= 1 || stride >= cols); }
bool any_stride_ok(int64_t s) { return s >= 0 && s <= kMaxStride; }
bool aligned(int64_t p, int64_t to) { return p % to == 0; }

// output scales [rows, groups]: no two of them in one place
bool scale_layout_ok(int64_t row, int64_t group, int64_t rows, int64_t ng) {
  if (!any_stride_ok(row) || !any_stride_ok(group)) return false;
  if (rows > 1 && row == 0) return false;
  if (ng > 1 && group == 0) return false;
  if (rows > 1 && ng > 1) return row > group * (ng - 1) || group > row * (rows - 1);
  return true;
}

}  // namespace

extern "C" {

int kcg_ops_load(int device) {
  return on_device(device, [](const HostHip*, const DeviceKernels&) { return (int)KCG_OK; });
}

int kcg_rmsnorm_quant(const kcg_rmsnorm_quant_args* p, int device, uint64_t stream) {
  if (!p) return bad("rmsnorm_quant: null argument");
  const int t = type_index(p->dtype);
  if (t < 0) return bad("rmsnorm_quant: x must be bfloat16, float16 or float32");
  if (p->weight_dtype != p->dtype && p->weight_dtype != KCG_DT_FLOAT32) return bad("rmsnorm_quant: the weight must have x's type or float32");
  if (!extent_ok(p->rows) || !extent_ok(p->cols)) return bad("rmsnorm_quant: rows and cols must be in [0, 2^30]");
  if (!(p->eps >= 0)) return bad("rmsnorm_quant: eps must not be negative");
  if (!p->residual != !p->residual_out) return bad("rmsnorm_quant: residual and residual_out go together");
  if (p->rows == 0 || p->cols == 0) return KCG_OK;
  if (!p->x || !p->weight || !p->q || !p->scale) return bad("rmsnorm_quant: null device pointer");
  const int es = type_bytes(p->dtype);
  if (!aligned(p->x, es) || !aligned(p->residual, es) || !aligned(p->residual_out, es) || !aligned(p->y, es) ||
      !aligned(p->weight, type_bytes(p->weight_dtype)) || !aligned(p->scale, 4))
    return bad("rmsnorm_quant: an address is not aligned to its elements");
  if (!aligned(p->q, 16) || (p->rows > 1 && !aligned(p->q_stride, 16))) return bad("rmsnorm_quant: rows of q must start on 16 bytes");
  if (!stride_ok(p->x_stride, p->cols, 1) || !stride_ok(p->q_stride, p->cols, p->rows) || (p->y && !stride_ok(p->y_stride, p->cols, p->rows)) ||
      (p->residual && (!stride_ok(p->residual_stride, p->cols, 1) || !stride_ok(p->residual_out_stride, p->cols, p->rows))))
    return bad("rmsnorm_quant: a row stride is negative or smaller than a row");
  if (!scale_layout_ok(p->scale_stride_row, p->scale_stride_group, p->rows, groups(p->cols))) return bad("rmsnorm_quant: scales overlap");
  NormArgs a = {(const void*)p->x, (const void*)p->residual, (void*)p->residual_out, (const void*)p->weight, (void*)p->y, (uint8_t*)p->q, (float*)p->scale,
                p->x_stride, p->residual_stride, p->residual_out_stride, p->y_stride, p->q_stride, p->scale_stride_row, p->scale_stride_group,
                (int)p->rows, (int)p->cols, p->weight_dtype == KCG_DT_FLOAT32, (float)p->eps};
  // threads per row: one vector of 8 each, up to 1024; two each up to 16384 columns; beyond, the row is read twice
  const int64_t nv = (p->cols + 7) / 8;
  const int v = nv <= 64 ? 0 : nv <= 128 ? 1 : nv <= 256 ? 2 : nv <= 512 ? 3 : nv <= 1024 ? 4 : nv <= 2048 ? 5 : 6;
  static const int threads[7] = {256, 128, 256, 512, 1024, 1024, 1024};
  const int64_t blocks = v == 0 ? (p->rows + 3) / 4 : p->rows;
  if (blocks * threads[v] > kMaxThreads) return bad("rmsnorm_quant: rows * cols is too large");
  return on_device(device, [&](const HostHip* hip, const DeviceKernels& k) {
    return launch(hip, k.fn[kNorm + t * 7 + v], (unsigned)blocks, 1, threads[v], 0, stream, &a);
  });
}

int kcg_swiglu_quant(const kcg_swiglu_quant_args* p, int device, uint64_t stream) {
  if (!p) return bad("swiglu_quant: null argument");
  const int t = type_index(p->dtype);
  if (t < 0) return bad("swiglu_quant: gate_up must be bfloat16, float16 or float32");
  if (!extent_ok(p->rows) || !extent_ok(p->cols)) return bad("swiglu_quant: rows and cols must be in [0, 2^30]");
  if (p->rows == 0 || p->cols == 0) return KCG_OK;
  if (!p->gate_up || !p->q || !p->scale) return bad("swiglu_quant: null device pointer");
  if (!aligned(p->gate_up, type_bytes(p->dtype)) || !aligned(p->scale, 4)) return bad("swiglu_quant: an address is not aligned to its elements");
  if (!aligned(p->q, 16) || (p->rows > 1 && !aligned(p->q_stride, 16))) return bad("swiglu_quant: rows of q must start on 16 bytes");
  if (!stride_ok(p->gate_up_stride, 2 * p->cols, 1) || !stride_ok(p->q_stride, p->cols, p->rows))
    return bad("swiglu_quant: a row stride is negative or smaller than a row");
  if (!scale_layout_ok(p->scale_stride_row, p->scale_stride_group, p->rows, groups(p->cols))) return bad("swiglu_quant: scales overlap");
  const int64_t threads = p->rows * groups(p->cols) * 16;
  if (threads > kMaxThreads - 256) return bad("swiglu_quant: rows * cols is too large");
  SwigluArgs a = {(const void*)p->gate_up, (uint8_t*)p->q, (float*)p->scale, p->gate_up_stride, p->q_stride, p->scale_stride_row, p->scale_stride_group,
                  (unsigned)p->rows, (int)p->cols};
  return on_device(device, [&](const HostHip* hip, const DeviceKernels& k) {
    return launch(hip, k.fn[kSwiglu + t], (unsigned)((threads + 255) / 256), 1, 256, 0, stream, &a);
  });
}

int kcg_matmul_fp8(const kcg_matmul_fp8_args* p, int device, uint64_t stream) {
  if (!p) return bad("matmul_fp8: null argument");
  const int t = type_index(p->c_dtype);
  if (t < 0) return bad("matmul_fp8: c must be bfloat16, float16 or float32");
  if (!extent_ok(p->m) || !extent_ok(p->n) || !extent_ok(p->k)) return bad("matmul_fp8: m, n and k must be in [0, 2^30]");
  if (p->m == 0 || p->n == 0) return KCG_OK;
  if (!p->c || (p->k > 0 && (!p->a || !p->a_scale || !p->b || !p->b_scale))) return bad("matmul_fp8: null device pointer");
  const int es = type_bytes(p->c_dtype);
  if (!aligned(p->c, es) || !aligned(p->a_scale, 4) || !aligned(p->b_scale, 4)) return bad("matmul_fp8: an address is not aligned to its elements");
  if (p->k > 0 && (!aligned(p->a, 16) || !aligned(p->b, 16) || (p->m > 1 && !aligned(p->a_stride, 16)) || (p->n > 1 && !aligned(p->b_stride, 16))))
    return bad("matmul_fp8: rows of a and b must start on 16 bytes");
  if (!stride_ok(p->a_stride, p->k, p->m) || !stride_ok(p->b_stride, p->k, p->n) || !stride_ok(p->c_stride, p->n, p->m))
    return bad("matmul_fp8: a row stride is negative or smaller than a row");
  if (!any_stride_ok(p->a_scale_stride_row) || !any_stride_ok(p->a_scale_stride_group) || !any_stride_ok(p->b_scale_stride_row) ||
      !any_stride_ok(p->b_scale_stride_group))
    return bad("matmul_fp8: a stride of the scales is negative");
  // a tile addresses its rows with 32-bit offsets from its first one
  if ((p->m > 1 && p->a_stride > (1 << 22)) || (p->n > 1 && p->b_stride > (1 << 22)) || (p->m > 1 && p->a_scale_stride_row > (1 << 20)) ||
      (p->n > 128 && p->b_scale_stride_row > (1 << 22)) || (p->k > 128 && (p->a_scale_stride_group > (1 << 22) || p->b_scale_stride_group > (1 << 22))))
    return bad("matmul_fp8: rows of a or b, or scales, are more than 2^22 elements apart, or rows of a_scale more than 2^20");
  MatmulArgs a = {(const uint8_t*)p->a, (const uint8_t*)p->b, (const float*)p->a_scale, (const float*)p->b_scale, (void*)p->c,
                  p->m > 1 ? p->a_stride : 0, p->n > 1 ? p->b_stride : 0, p->c_stride, p->m > 1 ? p->a_scale_stride_row : 0, p->a_scale_stride_group,
                  p->b_scale_stride_row, p->b_scale_stride_group, (int)p->m, (int)p->n, (int)p->k, (int)groups(p->k), 0, 0, 0};
  a.c_wide = aligned(p->c, 4 * es) && (p->m == 1 || aligned(p->c_stride, 4));
  const MatmulChoice c = choose_matmul(p->m, p->n, p->k, t);
  if (c.blocks * c.threads > kMaxThreads) return bad("matmul_fp8: m * n is too large");
  a.grid_m = c.grid_m;
  a.grid_n = c.grid_n;
  return on_device(device, [&](const HostHip* hip, const DeviceKernels& k) { return launch(hip, k.fn[c.fn], (unsigned)c.blocks, 1, c.threads, 0, stream, &a); });
}

int kcg_matmul_fp8_kernel(int64_t m, int64_t n, int64_t k, int64_t c_dtype, char* out, int out_len) {
  const int t = type_index(c_dtype);
  if (t < 0 || !extent_ok(m) || !extent_ok(n) || !extent_ok(k) || !out || out_len < 1) return bad("matmul_fp8_kernel: sizes in [0, 2^30], a 16 or 32-bit type, a buffer");
  try {
    const std::string s = m && n ? kernel_symbol(choose_matmul(m, n, k, t).fn) : "";
    snprintf(out, (size_t)out_len, "%s", s.c_str());
    return (int)s.size();
  } catch (...) {
    return KCG_ERR_ARGUMENT;
  }
}

int64_t kcg_moe_workspace_bytes(int64_t tokens, int64_t experts, int64_t topk, int64_t hidden, int64_t inter) {
  if (tokens < 0 || tokens > MOE_T) return bad("moe_layer: tokens must be in [0, 64] (this is the layer for a few tokens)");
  if (experts < 1 || experts > MOE_E) return bad("moe_layer: experts must be in [1, 512]");
  if (topk < 1 || topk > MOE_K || topk > experts) return bad("moe_layer: topk must be in [1, 16] and at most experts");
  if (hidden < 16 || hidden % 16 || hidden > (1 << 20) || inter < 16 || inter % 16 || inter > (1 << 20))
    return bad("moe_layer: hidden and inter must be multiples of 16, at most 2^20");
  return moe_plan(tokens, experts, topk, hidden, inter).bytes;
}

int kcg_moe_layer(const kcg_moe_layer_args* p, int device, uint64_t stream) {
  if (!p) return bad("moe_layer: null argument");
  const int64_t need = kcg_moe_workspace_bytes(p->tokens, p->experts, p->topk, p->hidden, p->inter);
  if (need < 0) return (int)need;
  int v;
  if (p->weight_dtype == KCG_DT_E4M3 && p->dtype == KCG_DT_BFLOAT16) v = 0;
  else if (p->weight_dtype == KCG_DT_E4M3 && p->dtype == KCG_DT_FLOAT16) v = 1;
  else if (p->weight_dtype == KCG_DT_BFLOAT16 && p->dtype == KCG_DT_BFLOAT16) v = 2;
  else return bad("moe_layer: weights in e4m3 with x in bfloat16 or float16, or both in bfloat16");
  if (p->tokens == 0) return KCG_OK;
  if (!p->x || !p->logits || !p->w13 || !p->w2 || !p->out || !p->ids || !p->probs || !p->workspace) return bad("moe_layer: null device pointer");
  if (v != 2 && (!p->w13_scale || !p->w2_scale)) return bad("moe_layer: e4m3 weights need their scales");
  if (p->workspace_bytes < need) return bad("moe_layer: the workspace is smaller than kcg_moe_workspace_bytes says");
  if (!aligned(p->x, 2) || !aligned(p->out, 2) || !aligned(p->logits, 4) || !aligned(p->ids, 4) || !aligned(p->probs, 4) || !aligned(p->w13_scale, 4) ||
      !aligned(p->w2_scale, 4))
    return bad("moe_layer: an address is not aligned to its elements");
  const int64_t wb = type_bytes(p->weight_dtype), per16 = 16 / wb;
  if (!aligned(p->w13, 16) || !aligned(p->w2, 16) || !aligned(p->workspace, 16) || !aligned(p->w13_stride_row, per16) ||
      !aligned(p->w2_stride_row, per16) || (p->experts > 1 && (!aligned(p->w13_stride_expert, per16) || !aligned(p->w2_stride_expert, per16))))
    return bad("moe_layer: the workspace and the rows of w13 and w2 must start on 16 bytes");
  if (!stride_ok(p->x_stride, p->hidden, 1) || !stride_ok(p->out_stride, p->hidden, p->tokens) || !any_stride_ok(p->logits_stride) ||
      !any_stride_ok(p->w13_stride_expert) || !any_stride_ok(p->w13_stride_row) || !any_stride_ok(p->w2_stride_expert) ||
      !any_stride_ok(p->w2_stride_row))
    return bad("moe_layer: a stride is negative, or rows of out overlap");
  const MoePlan m = moe_plan(p->tokens, p->experts, p->topk, p->hidden, p->inter);
  char* ws = (char*)p->workspace;
  MoeArgs a = {(const void*)p->x, (const float*)p->logits, (const void*)p->w13, (const void*)p->w2, (const float*)p->w13_scale, (const float*)p->w2_scale,
               (void*)p->out, (int32_t*)p->ids, (float*)p->probs, ws, ws + m.plane, (float*)(ws + 2 * m.plane), (int*)(ws + m.parts_at), (float*)(ws + m.y_at),
               p->x_stride, p->logits_stride, p->out_stride, p->w13_stride_expert, p->w13_stride_row, p->w2_stride_expert, p->w2_stride_row,
               (int)p->tokens, (int)p->experts, (int)p->topk, (int)p->hidden, (int)p->inter, (int)m.slots, p->renormalize != 0, 2, m.max_parts};
  // Waves that share 16 rows of the first product: as few as leave 4096 waves to the chip, two at least (64 tokens, 8 of 128
  // experts of 1024 x 4096: the call takes 339 with one, 303 with two, 326 with four, 365 with eight; one token, 8 of 64 experts
  // of 1024 x 2048: 33.5, 24.4, 19.7 and 19.3).
  const int64_t row_groups = p->inter / 16;
  while (a.split < UP_WAVES && row_groups * m.slots * a.split < 4096) a.split *= 2;
  const int per_block = UP_WAVES / a.split;
  return on_device(device, [&](const HostHip* hip, const DeviceKernels& k) {
    if (int rc = launch(hip, k.fn[kMoeUp + v], (unsigned)((row_groups + per_block - 1) / per_block), (unsigned)m.slots, UP_WAVES * 64, 0, stream, &a)) return rc;
    if (m.few)
      return launch(hip, k.fn[kMoeFew + v], (unsigned)(p->hidden / 16), 1, DOWN_WAVES * 64,
                    moe_partial_bytes(p->tokens) + (int)moe_h_bytes(p->tokens * p->topk, p->inter), stream, &a);
    if (int rc = launch(hip, k.fn[kMoeMany + 2 * (v == 2) + (m.per == 16)], (unsigned)((p->hidden + DOWN_MANY_COLS - 1) / DOWN_MANY_COLS), (unsigned)m.z, DOWN_MANY_WAVES * 64, 0,
                        stream, &a))
      return rc;
    return launch(hip, k.fn[kMoeCombine + (v == 1)], (unsigned)((p->hidden + 1023) / 1024), (unsigned)p->tokens, 256, 0, stream, &a);
  });
}

}  // extern "C"
