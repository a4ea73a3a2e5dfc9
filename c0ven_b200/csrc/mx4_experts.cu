// Products of MX rows in expert order with their experts' MX matrices (include/moe_layer.h: moe_mx4_product_device, moe_mx4_gate_up_device),
// on the tensor core's own 4-bit product: nothing is decoded.
//
// A work item is 128 rows of one expert's matrix (for gate_up 64 gate rows and the 64 up rows of the same features) times up to kTokens of
// the expert's rows. The matrix is the instruction's M side and the rows its N side, so a few rows cost a short instruction and what an item
// costs is bringing the matrix. Persistent CTAs, one an SM, take items in turn; items of one expert are neighbours.
//
// Roles of a CTA's ten warps: one thread brings codes by bulk-tensor copies, 256 values of the contraction a stage; four warps bring the scales,
// four stages (1,024 values: a sector of a row's scales) at a time in turn, word by word into the layout that the tensor core's copy reads
// (an expert's first row lies anywhere, so rows' scales cannot be laid out in advance); one lane issues scale copies and MMAs; four warps
// turn accumulators, of which there are two sets, into results.
//
// Every wait on an mbarrier is bounded: one that runs out raises the CTA's abort flag and the device's error word (moe_ops_status), the other
// waits return at once, and the CTA frees its tensor memory before it exits.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "mx4.cuh"
#include "mx4_mma.cuh"
#include "ops_common.h"
#include "tensor_map.h"

namespace moe {
namespace {

constexpr uint32_t kMaxExperts = 512;
constexpr uint32_t kRowsM = 128;        // matrix rows of an item
constexpr uint32_t kStageK = 256;       // values of the contraction a stage holds: 128 bytes of a row
constexpr uint32_t kScaleStages = 4;    // stages that one slot of scales covers
constexpr uint32_t kScaleSlots = 4;     // and as many warps fill them
constexpr uint32_t kBoxRows = 16;       // rows one copy of the rows' codes brings

// Barriers of the four epilogue warps alone. The second tells every one of them whether ok holds for all: they leave their loop together
// or not at all, so that none waits here for one that has left.
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

__device__ uint32_t g_gave_up;  // a wait ran out since moe_ops_status last asked

struct Mx4Args {
  const uint8_t *ws, *xs;   // scales of the matrices and the rows
  const int32_t *offsets;
  uint32_t E, N, K, R;
  uint32_t items_per_tile;  // items that share a tile of rows
  float limit;
  void *y;
  uint32_t bf16;
  uint8_t *hc, *hs;
};

// Shared memory of a CTA, for tiles of at most NT rows. Stages of codes; slots of scales, the matrix's and then the rows', eight pieces of 512
// bytes each; for gate_up the accumulators on their way to the quantiser; barriers; the experts' first rows and tiles.
template <bool GU, uint32_t NT>
struct Mx4Smem {
  static constexpr uint32_t kStages = 8;
  static constexpr uint32_t kStageBytes = (kRowsM + NT) * 128;
  static constexpr uint32_t kScales = kStages * kStageBytes;
  static constexpr uint32_t kSlotBytes = 2 * 8 * 512;
  static constexpr uint32_t kStaging = kScales + kScaleSlots * kSlotBytes;
  static constexpr uint32_t kStagingRow = kRowsM + 4;  // floats of a row of the tile, padded
  static constexpr uint32_t kBarriers = kStaging + (GU ? NT * kStagingRow * 4 : 0);
  static constexpr uint32_t kTables = kBarriers + 256;
  static constexpr uint32_t kBytes = kTables + 3 * (kMaxExperts + 1) * 4 + 1024;  // and room to align the base to 1024
  static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
  static_assert(NT <= 128, "the rows' scales are one piece a word");
};

constexpr uint32_t kThreads = 320;
enum : uint32_t { kCopyWarp = 0, kMmaWarp = 1, kScaleWarp = 2, kEpilogueWarp = 6 };

template <bool GU, uint32_t NT>
__global__ void __launch_bounds__(kThreads, 1) k_mx4_product(const __grid_constant__ Mx4Args a, const __grid_constant__ CUtensorMap wmap,
                                                             const __grid_constant__ CUtensorMap xmap) {
  using namespace tc;
  using SM = Mx4Smem<GU, NT>;
  constexpr uint32_t S = SM::kStages;
  constexpr uint32_t kScaleCols = 2 * NT;          // columns of the scales: 8 of the matrix's and 8 of the rows' a stage
  constexpr uint32_t kCols = kScaleCols + 16 * S <= 256 ? 256 : 512;
  static_assert(kScaleCols + 16 * S <= kCols, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  uint64_t *bars = (uint64_t *)(smem + SM::kBarriers);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty_bar = [&](uint32_t s) { return bar0 + 8 * (S + s); };
  auto scales_full = [&](uint32_t s) { return bar0 + 8 * (2 * S + s); };
  auto scales_empty = [&](uint32_t s) { return bar0 + 8 * (2 * S + kScaleSlots + s); };
  auto acc_full = [&](uint32_t b) { return bar0 + 8 * (2 * S + 2 * kScaleSlots + b); };
  auto acc_empty = [&](uint32_t b) { return bar0 + 8 * (2 * S + 2 * kScaleSlots + 2 + b); };
  static_assert(8 * (2 * S + 2 * kScaleSlots + 4) + 8 <= 256, "the barriers' room");
  uint32_t *tmem_slot = (uint32_t *)(bars + 2 * S + 2 * kScaleSlots + 4);
  volatile uint32_t *abort = tmem_slot + 1;
  uint32_t *first_row = (uint32_t *)(smem + SM::kTables), *end_row = first_row + kMaxExperts + 1, *first_tile = end_row + kMaxExperts + 1;
  uint32_t *error = &g_gave_up;

  if (tid == 0) {
    for (uint32_t s = 0; s < S; s++) mbar_init(full_bar(s), 1), mbar_init(empty_bar(s), 1);
    for (uint32_t s = 0; s < kScaleSlots; s++) mbar_init(scales_full(s), 1), mbar_init(scales_empty(s), 1);
    for (uint32_t b = 0; b < 2; b++) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 4);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(smem_u32(tmem_slot), kCols);
  dependents_may_launch(), wait_for_predecessors();
  // The experts' rows and tiles, summed up by one warp, 16 experts a lane. Offsets are held to 0 .. R and to their order.
  if (warp == kEpilogueWarp) {
    const uint32_t per = (a.E + 31) / 32, e0 = min(a.E, lane * per), e1 = min(a.E, e0 + per);
    auto row_of = [&](uint32_t e) { return a.offsets ? min((uint32_t)max(a.offsets[e], 0), a.R) : e ? a.R : 0u; };
    uint32_t sum = 0;
    for (uint32_t e = e0; e < e1; e++) {
      const uint32_t lo = row_of(e), hi = row_of(e + 1), n = hi > lo ? hi - lo : 0;
      first_row[e] = lo, end_row[e] = lo + n;
      sum += (n + NT - 1) / NT;
    }
    uint32_t before = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, before, off);
      if (lane >= (uint32_t)off) before += o;
    }
    before -= sum;
    for (uint32_t e = e0; e < e1; e++) {
      first_tile[e] = before;
      before += (end_row[e] - first_row[e] + NT - 1) / NT;
    }
    if (lane == 31) first_tile[a.E] = before;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t M = a.items_per_tile, K = a.K, F = a.N / 2, KT = (K + kStageK - 1) / kStageK;
  const uint32_t nitems = first_tile[a.E] * M;  // 2^24 / 32 + 512 tiles of 1,024 at most
  bool ok = true;

  struct Tile {
    uint32_t expert, start, count, m;
  };
  // Item i: tile i / M of the experts' tiles in order, and which of its M pieces of the matrix.
  auto tile_at = [&](uint32_t i) {
    const uint32_t t = i / M;
    uint32_t lo = 0, hi = a.E;  // the last expert whose first tile is at most t
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (first_tile[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    const uint32_t start = first_row[lo] + (t - first_tile[lo]) * NT;
    return Tile{lo, start, min(NT, end_row[lo] - start), i - t * M};
  };

  if (warp == kCopyWarp) {
    if (lane == 0) {
      uint32_t g = 0;  // stages used so far
      for (uint32_t i = blockIdx.x; i < nitems && ok; i += gridDim.x) {
        const Tile t = tile_at(i);
        const uint32_t boxes = (t.count + kBoxRows - 1) / kBoxRows;
        for (uint32_t it = 0; it < KT && ok; it++, g++) {
          const uint32_t s = g % S, use = g / S;
          if (use > 0) ok = mbar_wait(empty_bar(s), (use - 1) & 1, abort, error);
          if (!ok) break;
          const uint32_t at = smem_u32(smem + s * SM::kStageBytes), x0 = it * (kStageK / 2);
          mbar_arrive_expect(full_bar(s), kRowsM * 128 + boxes * kBoxRows * 128);
          if constexpr (GU) {
            tma_load_quants(at, &wmap, x0, t.m * 64, t.expert, full_bar(s));
            tma_load_quants(at + 64 * 128, &wmap, x0, F + t.m * 64, t.expert, full_bar(s));
          } else {
            tma_load_quants(at, &wmap, x0, t.m * kRowsM, t.expert, full_bar(s));
          }
          for (uint32_t b = 0; b < boxes; b++) tma_load_quants(at + (kRowsM + b * kBoxRows) * 128, &xmap, x0, t.start + b * kBoxRows, 0, full_bar(s));
        }
      }
      if (!ok) {
        // Copies already issued may still be on their way: give them time to land before the CTA leaves.
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {
        }
      }
    }
  } else if (warp >= kScaleWarp && warp < kScaleWarp + kScaleSlots) {
    // A slot of scales by a warp: four rows' eight words an instruction, so that a row's 32 bytes are one request.
    const uint32_t mine = warp - kScaleWarp, srow = mx_scale_row_bytes(K), nb = K / kMxBlock, slots = (KT + kScaleStages - 1) / kScaleStages;
    const uint32_t word = lane % 8, at = smem_u32(smem + SM::kScales + mine * SM::kSlotBytes) + word * 512;
    uint32_t g = 0;  // slots filled so far, by all
    for (uint32_t i = blockIdx.x; i < nitems && ok; i += gridDim.x) {
      const Tile t = tile_at(i);
      for (uint32_t j = 0; j < slots && ok; j++, g++) {
        if (g % kScaleSlots != mine) continue;
        const uint32_t use = g / kScaleSlots;
        if (use > 0) ok = mbar_wait_warp(scales_empty(mine), (use - 1) & 1, abort, error);
        if (!ok) break;
        const uint32_t b0 = j * (kScaleStages * kStageK / kMxBlock) + 4 * word, n = b0 < nb ? min(4u, nb - b0) : 0u;
        for (uint32_t r = lane / 8; r < kRowsM; r += 4) {
          uint32_t row = GU ? (r < 64 ? t.m * 64 + r : F + t.m * 64 + r - 64) : t.m * kRowsM + r;
          const uint32_t have = row < a.N ? n : 0;
          copy_word(at + 16 * (r % 32) + 4 * (r / 32), have ? a.ws + ((uint64_t)t.expert * a.N + row) * srow + b0 : a.ws, have);
        }
        for (uint32_t r = lane / 8; r < ((t.count + 3) & ~3u); r += 4) {
          const uint32_t have = r < t.count ? n : 0;
          copy_word(at + 8 * 512 + 16 * (r % 32) + 4 * (r / 32), have ? a.xs + (uint64_t)(t.start + r) * srow + b0 : a.xs, have);
        }
        copy_words_wait();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(scales_full(mine));
      }
    }
  } else if (warp == kMmaWarp) {
    const uint32_t leader = elect_leader();
    uint32_t g = 0, gs = 0, li = 0;
    for (uint32_t i = blockIdx.x; i < nitems && ok; i += gridDim.x, li++) {
      const Tile t = tile_at(i);
      const uint32_t n = (t.count + 15) & ~15u, b = li & 1, acc = tmem_base + b * NT;
      const uint32_t d0 = mx4_instr_desc(n, kRowsM, 0), d2 = mx4_instr_desc(n, kRowsM, 2);
      if (li > 1) ok = mbar_wait_warp(acc_empty(b), (li / 2 - 1) & 1, abort, error);
      for (uint32_t it = 0; it < KT && ok; it++, g++) {
        const uint32_t s = g % S, slot = gs % kScaleSlots, sub = it % kScaleStages;
        if (sub == 0) ok = mbar_wait_warp(scales_full(slot), (gs / kScaleSlots) & 1, abort, error);
        if (ok) ok = mbar_wait_warp(full_bar(s), (g / S) & 1, abort, error);
        if (!ok) break;
        tc_fence_after();
        const uint32_t stage = smem_u32(smem + s * SM::kStageBytes), rows = stage + kRowsM * 128;
        const uint32_t sc = smem_u32(smem + SM::kScales + slot * SM::kSlotBytes) + 2 * sub * 512, ta = tmem_base + kScaleCols + 16 * s, tb = ta + 8;
        // The stage's columns of scales are its own: the MMAs that read them last are done, for the stage was empty again.
        copy_scales(leader, ta, sc), copy_scales(leader, ta + 4, sc + 512);
        copy_scales(leader, tb, sc + 8 * 512), copy_scales(leader, tb + 4, sc + 9 * 512);
        const uint32_t steps = min(4u, (K - it * kStageK + 63) / 64);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
          if (k < steps)
            mma_mx4(leader, acc, smem_desc_sw128(stage + 32 * k), smem_desc_sw128(rows + 32 * k), k % 2 ? d2 : d0, ta + 4 * (k / 2), tb + 4 * (k / 2), (it | k) != 0);
        mma_commit(leader, empty_bar(s));
        if (sub == kScaleStages - 1 || it == KT - 1) mma_commit(leader, scales_empty(slot)), gs++;
      }
      if (!ok) break;
      mma_commit(leader, acc_full(b));
    }
  } else if (warp >= kEpilogueWarp) {
    // Warp w reads tensor memory's lanes 32 (w % 4) ...
    const uint32_t q = warp % 4;
    uint32_t li = 0;
    for (uint32_t i = blockIdx.x; i < nitems && ok; i += gridDim.x, li++) {
      const Tile t = tile_at(i);
      const uint32_t b = li & 1, from = tmem_base + ((32 * q) << 16) + b * NT;
      ok = mbar_wait_warp(acc_full(b), (li / 2) & 1, abort, error);
      if constexpr (GU) ok = epilogue_all(ok);  // the staging room's item before has been read, too
      if (!ok) break;
      tc_fence_after();
      if constexpr (!GU) {
        const uint32_t n = t.m * kRowsM + 32 * q + lane;
        for (uint32_t c = 0; c < t.count; c += 16) {
          uint32_t v[16];
          tmem_ld16(from + c, v);
          tmem_ld_wait16(v);
          const uint64_t at = (uint64_t)(t.start + c) * a.N + n;
#pragma unroll
          for (uint32_t j = 0; j < 16; j++) {
            if (c + j >= t.count || n >= a.N) continue;
            if (a.bf16)
              ((__nv_bfloat16 *)a.y)[at + (uint64_t)j * a.N] = __float2bfloat16_rn(__uint_as_float(v[j]));
            else
              ((__half *)a.y)[at + (uint64_t)j * a.N] = __float2half_rn(__uint_as_float(v[j]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(b));
      } else {
        // Through shared memory, a row of the tile its 64 gate and 64 up products, to threads of eight features each.
        float *st = (float *)(smem + SM::kStaging);
        for (uint32_t c = 0; c < t.count; c += 16) {
          uint32_t v[16];
          tmem_ld16(from + c, v);
          tmem_ld_wait16(v);
#pragma unroll
          for (uint32_t j = 0; j < 16; j++) st[(c + j) * SM::kStagingRow + 32 * q + lane] = __uint_as_float(v[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(b));
        epilogue_sync();
        const uint32_t f = (tid % 8) * 8, hrow = mx_scale_row_bytes(F), at = t.m * 64 + f;
        for (uint32_t r0 = 0; r0 < t.count; r0 += 16) {
          const uint32_t r = r0 + (tid - 32 * kEpilogueWarp) / 8;
          float h[8];
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float *p = st + min(r, NT - 1) * SM::kStagingRow + f + j;
            h[j] = swiglu(p[0], p[64], a.limit);
            m = max(m, __float_as_uint(h[j]) & 0x7FFFFFFFu);
          }
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const uint32_t scale = mx_scale_of(m);
          const float inv = mx_inverse(scale);
#pragma unroll
          for (int j = 0; j < 8; j++) h[j] *= inv;
          if (r >= t.count || at >= F) continue;
          const uint64_t row = t.start + r;
          *(uint32_t *)(a.hc + row * (F / 2) + at / 2) = scale == 255 ? 0u : mx_codes8(h);
          if (tid % 4 == 0) a.hs[row * hrow + at / kMxBlock] = (uint8_t)scale;
          if (tid % 4 == 0 && at + kMxBlock == F)
            for (uint32_t s = F / kMxBlock; s < hrow; s++) a.hs[row * hrow + s] = 0;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem_base, kCols);
  }
}

template <bool GU, uint32_t NT>
void launch_product(const Mx4Args &args, const uint8_t *wc, const uint8_t *xc, cudaStream_t st) {
  Mx4Args a = args;
  int device = 0;
  CUDA_OK(cudaGetDevice(&device));
  constexpr size_t smem = Mx4Smem<GU, NT>::kBytes;
  static std::atomic<uint32_t> done{0};
  CUDA_OK(ensure_dynamic_smem(k_mx4_product<GU, NT>, smem, done, device));
  int sms = 0;
  CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  a.items_per_tile = GU ? (a.N / 2 + 63) / 64 : (a.N + kRowsM - 1) / kRowsM;
  const uint64_t most = ((uint64_t)a.R / NT + std::min(a.E, a.R)) * a.items_per_tile;  // items there can be
  const CUtensorMap wmap = make_codes_map(wc, a.K / 2, a.N, a.E, GU ? 64 : kRowsM), xmap = make_codes_map(xc, a.K / 2, a.R, 1, kBoxRows);
  CUDA_OK(launch_kernel(true, k_mx4_product<GU, NT>, dim3((unsigned)std::min<uint64_t>(most, (uint64_t)sms)), dim3(kThreads), smem, st, a, wmap, xmap));
}

Mx4Args arguments(const moe_mx4_weights *w, const void *scales, uint32_t R, const int32_t *offsets) {
  need(w != nullptr, "weights are required");
  need(w->n_experts >= 1 && w->n_experts <= kMaxExperts, "n_experts must be 1 .. 512");
  need(w->n_out >= 32 && w->n_out % 32 == 0 && w->n_out <= kMxMaxValues, "n_out must be a multiple of 32, 32 .. 65536");
  need(w->n_in >= 32 && w->n_in % 32 == 0 && w->n_in <= kMxMaxValues, "n_in must be a multiple of 32, 32 .. 65536");
  need(w->reserved == 0, "reserved must be 0");
  need(offsets || w->n_experts == 1, "offsets are required for more than one expert");
  need(R <= 1u << 24, "R must be at most 2^24");
  Mx4Args a{};
  a.ws = (const uint8_t *)w->scales_dev, a.xs = (const uint8_t *)scales;
  a.offsets = offsets, a.E = w->n_experts, a.N = w->n_out, a.K = w->n_in, a.R = R;
  return a;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API moe_status moe_mx4_product_device(const moe_mx4_weights *w, const void *codes_dev, const void *scales_dev, uint32_t R,
                                          const int32_t *offsets_dev, void *y_dev, uint32_t y_type, void *stream) {
  return ops_call([&] {
    need(y_type == MOE_TYPE_F16 || y_type == MOE_TYPE_BF16, "y_type must be MOE_TYPE_F16 or MOE_TYPE_BF16");
    Mx4Args a = arguments(w, scales_dev, R, offsets_dev);
    if (R == 0) return;
    need_device({{w->codes_dev, "weight codes", 16}, {a.ws, "weight scales", 4}, {codes_dev, "codes", 16}, {a.xs, "scales", 4}, {a.offsets, "offsets", 4, true}, {y_dev, "y", 16}});
    a.y = y_dev, a.bf16 = y_type == MOE_TYPE_BF16;
    launch_product<false, 32>(a, (const uint8_t *)w->codes_dev, (const uint8_t *)codes_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_mx4_gate_up_device(const moe_mx4_weights *w, const void *codes_dev, const void *scales_dev, uint32_t R,
                                          const int32_t *offsets_dev, float swiglu_limit, void *h_codes_dev, void *h_scales_dev, void *stream) {
  return ops_call([&] {
    need(!(swiglu_limit < 0.0f) && swiglu_limit - swiglu_limit == 0.0f, "swiglu_limit must be 0 or a positive number");
    Mx4Args a = arguments(w, scales_dev, R, offsets_dev);
    need(a.N % 64 == 0, "gate and up rows together must be a multiple of 64");
    if (R == 0) return;
    need_device({{w->codes_dev, "weight codes", 16}, {a.ws, "weight scales", 4}, {codes_dev, "codes", 16}, {a.xs, "scales", 4}, {a.offsets, "offsets", 4, true},
                 {h_codes_dev, "h codes", 16}, {h_scales_dev, "h scales", 4}});
    a.limit = swiglu_limit, a.hc = (uint8_t *)h_codes_dev, a.hs = (uint8_t *)h_scales_dev;
    launch_product<true, 32>(a, (const uint8_t *)w->codes_dev, (const uint8_t *)codes_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_ops_status(uint32_t timeout_ms, void *stream) {
  return ops_call([&] {
    Stream::wait_on((cudaStream_t)stream, timeout_ms);
    uint32_t gave_up = 0, none = 0;
    CUDA_OK(cudaMemcpyFromSymbol(&gave_up, g_gave_up, sizeof gave_up));
    if (!gave_up) return;
    CUDA_OK(cudaMemcpyToSymbol(g_gave_up, &none, sizeof none));
    throw Timeout("a product gave up waiting for its copies or its products: its results are not to be used");
  });
}

}  // extern "C"
