// Products of MX rows in expert order with their experts' MX matrices (include/moe_layer.h: moe_mx4_product_device, moe_mx4_gate_up_device),
// on the tensor core's own 4-bit product: nothing is decoded.
//
// A work item is 128 rows of one expert's matrix for each CTA that works on it (for gate_up 64 gate rows and the 64 up rows of the same
// features) times up to NT of the expert's rows. The matrix is the instruction's M side and the rows its N side, so a few rows cost a
// short instruction and what an item costs is bringing the matrix. Persistent units (a CTA, or a pair of CTAs on two SMs that share the rows:
// tcgen05's cta_group::2) take items in turn; items of one expert are neighbours.
//
// Roles of a CTA's warps: one thread brings codes by bulk-tensor copies, 256 values of the contraction a stage; four warps bring the scales,
// four stages (1,024 values: a sector of a row's scales) at a time in turn, word by word into the layout that the tensor core's copy reads
// (an expert's first row lies anywhere, so rows' scales cannot be laid out in advance); one lane (of a pair's first CTA) issues scale copies and
// MMAs; groups of four warps turn accumulators, of which there are two sets, into results.
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
constexpr uint32_t kRowsM = 128;        // matrix rows a CTA takes
constexpr uint32_t kStageK = 256;       // values of the contraction a stage holds: 128 bytes of a row
constexpr uint32_t kScaleStages = 4;    // stages that one slot of scales covers
constexpr uint32_t kBoxRows = 16;       // rows one copy of the rows' codes brings
constexpr uint32_t kChunk = 16;         // rows an epilogue warp turns at a time

// Barriers of a group of four epilogue warps alone. The second tells every one of them whether ok holds for all: they leave their loop together
// or not at all, so that none waits here for one that has left.
__device__ __forceinline__ void group_sync(uint32_t group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
__device__ __forceinline__ bool group_all(uint32_t group, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(1 + group)
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

// A form of the kernel: CTAs a unit has, and the most rows of a tile. Its shared memory: stages of codes; slots of scales, the matrix's and then
// the rows', eight words of every row each; for gate_up the accumulators on their way to the quantiser, two chunks a group; barriers; the
// experts' first and last rows and first tiles.
template <bool GU, uint32_t CTAS, uint32_t NT>
struct Mx4Form {
  static constexpr uint32_t kGroups = CTAS;  // of four epilogue warps
  static constexpr uint32_t kThreads = 32 * (6 + 4 * kGroups);
  static constexpr uint32_t kStages = CTAS == 2 ? 5 : 8;
  static constexpr uint32_t kStageBytes = (kRowsM + NT / CTAS) * 128;
  static constexpr uint32_t kScaleSlots = CTAS == 2 ? 3 : 4;
  static constexpr uint32_t kRowPieces = (NT + 127) / 128;  // 512-byte pieces a word of the rows' scales takes
  static constexpr uint32_t kScales = kStages * kStageBytes;
  static constexpr uint32_t kSlotBytes = (1 + kRowPieces) * 8 * 512;
  static constexpr uint32_t kStaging = kScales + kScaleSlots * kSlotBytes;
  static constexpr uint32_t kStagingRow = kRowsM + 4;  // floats of a row of a chunk, padded
  static constexpr uint32_t kStagingBytes = kChunk * kStagingRow * 4;
  static constexpr uint32_t kBarriers = kStaging + (GU ? 2 * kGroups * kStagingBytes : 0);
  static constexpr uint32_t kTables = kBarriers + 256;
  static constexpr uint32_t kBytes = kTables + 3 * (kMaxExperts + 1) * 4 + 1024;  // and room to align the base to 1024
  static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
  // Tensor memory: two accumulators, then the scales of kScaleRing stages.
  static constexpr uint32_t kScaleCols = 8 + 8 * kRowPieces;
  static constexpr uint32_t kScaleRing = CTAS == 2 ? 2 : kStages;
  static constexpr uint32_t kUsedCols = 2 * NT + kScaleRing * kScaleCols;
  static constexpr uint32_t kCols = kUsedCols <= 256 ? 256 : 512;
  static_assert(kUsedCols <= kCols, "tensor memory");
};

enum : uint32_t { kCopyWarp = 0, kMmaWarp = 1, kScaleWarp = 2, kEpilogueWarp = 6 };

// Rows a tile of an expert's n rows has: the tiles of a few share them evenly (which 16 rows a tile can be off by leaves no tile empty up to
// eight tiles of 224).
template <uint32_t NT>
__device__ __forceinline__ uint32_t tile_rows(uint32_t n) {
  const uint32_t tiles = (n + NT - 1) / NT;
  return NT >= 128 && tiles > 1 && tiles <= 8 ? ((n + tiles - 1) / tiles + 15) & ~15u : NT;
}

template <bool GU, uint32_t CTAS, uint32_t NT>
__global__ void __launch_bounds__(Mx4Form<GU, CTAS, NT>::kThreads, 1) k_mx4_product(const __grid_constant__ Mx4Args a, const __grid_constant__ CUtensorMap wmap,
                                                                                    const __grid_constant__ CUtensorMap xmap) {
  using namespace tc;
  using SM = Mx4Form<GU, CTAS, NT>;
  constexpr uint32_t S = SM::kStages, SL = SM::kScaleSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = CTAS == 2 ? cluster_ctarank() : 0, unit = blockIdx.x / CTAS, nunits = gridDim.x / CTAS;
  uint64_t *bars = (uint64_t *)(smem + SM::kBarriers);
  // Barriers: stages full, empty; scales full, empty; accumulators full, empty. Of a pair the first CTA's "full" of stages and scales and "empty"
  // of accumulators take both CTAs' arrivals.
  constexpr uint32_t kEmpty = S, kScFull = 2 * S, kScEmpty = kScFull + SL, kAccFull = kScEmpty + SL, kAccEmpty = kAccFull + 2, kBars = kAccEmpty + 2;
  static_assert(8 * kBars + 8 <= 256, "the barriers' room");
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](uint32_t i) { return bar0 + 8 * i; };
  uint32_t *tmem_slot = (uint32_t *)(bars + kBars);
  volatile uint32_t *abort = tmem_slot + 1;
  uint32_t *first_row = (uint32_t *)(smem + SM::kTables), *end_row = first_row + kMaxExperts + 1, *first_tile = end_row + kMaxExperts + 1;
  uint32_t *error = &g_gave_up;

  if (tid == 0) {
    for (uint32_t s = 0; s < S; s++) mbar_init(bar(s), CTAS), mbar_init(bar(kEmpty + s), 1);
    for (uint32_t s = 0; s < SL; s++) mbar_init(bar(kScFull + s), CTAS), mbar_init(bar(kScEmpty + s), 1);
    for (uint32_t b = 0; b < 2; b++) mbar_init(bar(kAccFull + b), 1), mbar_init(bar(kAccEmpty + b), CTAS * 4 * SM::kGroups);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    if constexpr (CTAS == 2)
      tmem_alloc_pair(smem_u32(tmem_slot), SM::kCols);
    else
      tmem_alloc(smem_u32(tmem_slot), SM::kCols);
  }
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
  if constexpr (CTAS == 2) cluster_sync();  // the other CTA's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t M = a.items_per_tile, K = a.K, F = a.N / 2, KT = (K + kStageK - 1) / kStageK;
  const uint32_t nitems = first_tile[a.E] * M;  // 2^24 / 32 + 512 tiles of 1,024 at most
  const uint32_t lead0 = CTAS == 2 ? map_to_cta(bar0, 0) : bar0;  // the first CTA's barriers as this CTA names them
  auto lead = [&](uint32_t i) { return lead0 + 8 * i; };
  auto arrive_lead = [&](uint32_t i) {
    if constexpr (CTAS == 2)
      mbar_arrive_cluster(lead(i));
    else
      mbar_arrive(lead(i));
  };
  bool ok = true;

  // row0: the first of this CTA's matrix rows, or of its features.
  struct Tile {
    uint32_t expert, start, count, row0;
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
    const uint32_t per = tile_rows<NT>(end_row[lo] - first_row[lo]), start = first_row[lo] + (t - first_tile[lo]) * per;
    return Tile{lo, start, min(per, end_row[lo] - start), ((i - t * M) * CTAS + rank) * (GU ? kRowsM / 2 : kRowsM)};
  };

  if (warp == kCopyWarp) {
    if (lane == 0) {
      uint32_t s = 0, phase = 1;  // of the stage's "empty": the first round finds it so
      for (uint32_t i = unit; i < nitems && ok; i += nunits) {
        const Tile t = tile_at(i);
        // A CTA of a pair brings its half of the rows the instruction takes, which are rounded up to 16.
        const uint32_t half = ((t.count + 15) & ~15u) / CTAS, x_row = t.start + rank * half, boxes = (half + kBoxRows - 1) / kBoxRows;
        for (uint32_t it = 0; it < KT && ok; it++) {
          ok = mbar_wait(bar(kEmpty + s), phase, abort, error);
          if (!ok) break;
          const uint32_t at = smem_u32(smem + s * SM::kStageBytes), x0 = it * (kStageK / 2);
          auto copy = [&](uint32_t dst, const CUtensorMap *map, uint32_t y, uint32_t z) {
            if constexpr (CTAS == 2)
              tma_load_codes_pair(dst, map, x0, y, z, lead(s));
            else
              tma_load_quants(dst, map, x0, y, z, lead(s));
          };
          if constexpr (CTAS == 2)
            mbar_arrive_expect_cluster(lead(s), kRowsM * 128 + boxes * kBoxRows * 128);
          else
            mbar_arrive_expect(lead(s), kRowsM * 128 + boxes * kBoxRows * 128);
          copy(at, &wmap, t.row0, t.expert);
          if constexpr (GU) copy(at + 64 * 128, &wmap, F + t.row0, t.expert);
          for (uint32_t b = 0; b < boxes; b++) copy(at + (kRowsM + b * kBoxRows) * 128, &xmap, x_row + b * kBoxRows, 0);
          if (++s == S) s = 0, phase ^= 1;
        }
      }
      if (!ok) {
        // Copies already issued may still be on their way: give them time to land before the CTA leaves.
        const long long t0 = clock64();
        while (clock64() - t0 < 400000) {
        }
      }
    }
  } else if (warp >= kScaleWarp && warp < kScaleWarp + SL) {
    // A slot of scales by a warp: four rows' eight words an instruction, so that a row's 32 bytes are one request.
    const uint32_t mine = warp - kScaleWarp, srow = mx_scale_row_bytes(K), nb = K / kMxBlock, slots = (KT + kScaleStages - 1) / kScaleStages;
    const uint32_t word = lane % 8, slot = smem_u32(smem + SM::kScales + mine * SM::kSlotBytes);
    const uint32_t at = slot + word * 512, x_at = slot + 8 * 512 + word * SM::kRowPieces * 512;
    uint32_t turn = 0, phase = 1;  // whose turn the next slot is
    for (uint32_t i = unit; i < nitems && ok; i += nunits) {
      const Tile t = tile_at(i);
      for (uint32_t j = 0; j < slots && ok; j++, turn = turn == SL - 1 ? 0 : turn + 1) {
        if (turn != mine) continue;
        ok = mbar_wait_warp(bar(kScEmpty + mine), phase, abort, error);
        if (!ok) break;
        phase ^= 1;
        const uint32_t b0 = j * (kScaleStages * kStageK / kMxBlock) + 4 * word, n = b0 < nb ? min(4u, nb - b0) : 0u;
        for (uint32_t r = lane / 8; r < kRowsM; r += 4) {
          const uint32_t row = GU ? (r < 64 ? t.row0 + r : F + t.row0 + r - 64) : t.row0 + r, have = row < a.N ? n : 0;
          copy_word(at + 16 * (r % 32) + 4 * (r / 32), have ? a.ws + ((uint64_t)t.expert * a.N + row) * srow + b0 : a.ws, have);
        }
        for (uint32_t r = lane / 8; r < ((t.count + 3) & ~3u); r += 4) {
          const uint32_t have = r < t.count ? n : 0;
          copy_word(x_at + r / 128 * 512 + 16 * (r % 32) + 4 * (r / 32 % 4), have ? a.xs + (uint64_t)(t.start + r) * srow + b0 : a.xs, have);
        }
        copy_words_wait();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive_lead(kScFull + mine);
      }
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint32_t leader = elect_leader();
      auto commit = [&](uint32_t i) {
        if constexpr (CTAS == 2)
          mma_commit_pair(leader, bar(i), 3);
        else
          mma_commit(leader, bar(i));
      };
      uint32_t s = 0, phase = 0, slot = 0, slot_phase = 0, ring = 0, b = 0, acc_phase = 1;
      uint32_t old = S - SM::kScaleRing % S, old_phase = 1;  // the stage whose scales the ring's next columns held, kScaleRing stages ago
      for (uint32_t i = unit; i < nitems && ok; i += nunits) {
        const Tile t = tile_at(i);
        const uint32_t n = (t.count + 15) & ~15u, acc = tmem_base + b * NT;
        const uint32_t d0 = mx4_instr_desc(n, CTAS * kRowsM, 0), d2 = mx4_instr_desc(n, CTAS * kRowsM, 2);
        ok = mbar_wait_warp(bar(kAccEmpty + b), acc_phase, abort, error);
        for (uint32_t it = 0; it < KT && ok; it++) {
          const uint32_t sub = it % kScaleStages;
          if (sub == 0) ok = mbar_wait_warp(bar(kScFull + slot), slot_phase, abort, error);
          if (ok) ok = mbar_wait_warp(bar(s), phase, abort, error);
          // The columns this stage's scales go to are free when the MMAs that read them are done: with as many columns as stages they are,
          // for the stage was empty again; else the commit after those MMAs says so.
          if constexpr (SM::kScaleRing < S)
            if (ok) ok = mbar_wait_warp(bar(kEmpty + old % S), old_phase, abort, error);
          if (!ok) break;
          tc_fence_after();
          const uint32_t stage = smem_u32(smem + s * SM::kStageBytes), rows = stage + kRowsM * 128;
          const uint32_t sc = smem_u32(smem + SM::kScales + slot * SM::kSlotBytes) + 2 * sub * 512;
          const uint32_t sx = smem_u32(smem + SM::kScales + slot * SM::kSlotBytes) + 8 * 512 + 2 * sub * SM::kRowPieces * 512;
          const uint32_t ta = tmem_base + 2 * NT + ring * SM::kScaleCols, tb = ta + 8;
          copy_scales<CTAS>(leader, ta, sc), copy_scales<CTAS>(leader, ta + 4, sc + 512);
#pragma unroll
          for (uint32_t p = 0; p < 2 * SM::kRowPieces; p++) copy_scales<CTAS>(leader, tb + 4 * p, sx + 512 * p);
          const uint32_t steps = min(4u, (K - it * kStageK + 63) / 64);
#pragma unroll
          for (uint32_t k = 0; k < 4; k++)
            if (k < steps)
              mma_mx4<CTAS>(leader, acc, smem_desc_sw128(stage + 32 * k), smem_desc_sw128(rows + 32 * k), k % 2 ? d2 : d0, ta + 4 * (k / 2),
                            tb + 4 * SM::kRowPieces * (k / 2), (it | k) != 0);
          commit(kEmpty + s);
          if (sub == kScaleStages - 1 || it == KT - 1) {
            commit(kScEmpty + slot);
            if (++slot == SL) slot = 0, slot_phase ^= 1;
          }
          if (++s == S) s = 0, phase ^= 1;
          if (++ring == SM::kScaleRing) ring = 0;
          if (++old == S) old = 0, old_phase ^= 1;
        }
        if (!ok) break;
        commit(kAccFull + b);
        acc_phase ^= b, b ^= 1;
      }
    }
  } else if (warp >= kEpilogueWarp) {
    // Warp w reads tensor memory's lanes 32 (w % 4) ...; the groups take chunks of 16 rows in turn.
    const uint32_t q = warp % 4, group = (warp - kEpilogueWarp) / 4;
    uint32_t b = 0, phase = 0;
    [[maybe_unused]] uint32_t turn = 0;
    for (uint32_t i = unit; i < nitems && ok; i += nunits) {
      const Tile t = tile_at(i);
      const uint32_t from = tmem_base + ((32 * q) << 16) + b * NT;
      ok = mbar_wait_warp(bar(kAccFull + b), phase, abort, error);
      if constexpr (GU) ok = group_all(group, ok);
      if (!ok) break;
      tc_fence_after();
      if constexpr (!GU) {
        const uint32_t n = t.row0 + 32 * q + lane;
        for (uint32_t c = group * kChunk; c < t.count; c += SM::kGroups * kChunk) {
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
      } else {
        // Through shared memory, a row of the chunk its 64 gate and 64 up products, to threads of eight features each. Of a group's two
        // chunks there the one is written while another warp may still read the other; past the barrier all have left it.
        const uint32_t f = (tid % 8) * 8, hrow = mx_scale_row_bytes(F), at = t.row0 + f, r = (tid / 8) % 16;
        for (uint32_t c = group * kChunk; c < t.count; c += SM::kGroups * kChunk, turn ^= 1) {
          float *st = (float *)(smem + SM::kStaging + (2 * group + turn) * SM::kStagingBytes);
          uint32_t v[16];
          tmem_ld16(from + c, v);
          tmem_ld_wait16(v);
#pragma unroll
          for (uint32_t j = 0; j < 16; j++) st[j * SM::kStagingRow + 32 * q + lane] = __uint_as_float(v[j]);
          group_sync(group);
          float h[8];
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float *p = st + r * SM::kStagingRow + f + j;
            h[j] = swiglu(p[0], p[64], a.limit);
            m = max(m, __float_as_uint(h[j]) & 0x7FFFFFFFu);
          }
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const uint32_t scale = mx_scale_of(m);
          const float inv = mx_inverse(scale);
#pragma unroll
          for (int j = 0; j < 8; j++) h[j] *= inv;
          if (c + r >= t.count || at >= F) continue;
          const uint64_t row = t.start + c + r;
          *(uint32_t *)(a.hc + row * (F / 2) + at / 2) = scale == 255 ? 0u : mx_codes8(h);
          if (tid % 4 == 0) a.hs[row * hrow + at / kMxBlock] = (uint8_t)scale;
          if (tid % 4 == 0 && at + kMxBlock == F)
            for (uint32_t s = F / kMxBlock; s < hrow; s++) a.hs[row * hrow + s] = 0;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_lead(kAccEmpty + b);
      phase ^= b, b ^= 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();  // neither CTA leaves while the other may still read its shared memory or write its tensor memory
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CTAS == 2)
      tmem_free_pair(tmem_base, SM::kCols);
    else
      tmem_free(tmem_base, SM::kCols);
  }
}

template <bool GU, uint32_t CTAS, uint32_t NT>
void launch_product(const Mx4Args &args, const void *wc, const void *xc, cudaStream_t st) {
  using Form = Mx4Form<GU, CTAS, NT>;
  constexpr auto kernel = k_mx4_product<GU, CTAS, NT>;
  Mx4Args a = args;
  int device = 0;
  CUDA_OK(cudaGetDevice(&device));
  constexpr size_t smem = Form::kBytes;
  static std::atomic<uint32_t> done{0};
  CUDA_OK(ensure_dynamic_smem(kernel, smem, done, device));
  uint32_t units = 0;
  if constexpr (CTAS == 2) {
    CUDA_OK(max_pairs<kernel>(Form::kThreads, smem, device, units));
  } else {
    int sms = 0;
    CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    units = (uint32_t)sms;
  }
  const uint32_t rows = CTAS * (GU ? kRowsM / 2 : kRowsM), all = GU ? a.N / 2 : a.N;
  a.items_per_tile = (all + rows - 1) / rows;
  const uint64_t most = ((uint64_t)a.R / NT + std::min(a.E, a.R)) * a.items_per_tile;  // items there can be
  const CUtensorMap wmap = make_codes_map(wc, a.K / 2, a.N, a.E, GU ? 64 : kRowsM), xmap = make_codes_map(xc, a.K / 2, a.R, 1, kBoxRows);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension, at[1].val.clusterDim = {CTAS, 1, 1};
  cfg.gridDim = dim3(CTAS * (unsigned)std::min<uint64_t>(most, units)), cfg.blockDim = dim3(Form::kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cfg.attrs = at, cfg.numAttrs = CTAS;  // a single CTA is no cluster
  CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a, wmap, xmap));
}

// Tiles of 224 rows by pairs of CTAs, or of 32 by single ones.
template <bool GU>
void launch(const Mx4Args &a, const void *wc, const void *xc, cudaStream_t st) {
  if (a.R > 32ull * a.E)
    launch_product<GU, 2, 224>(a, wc, xc, st);
  else
    launch_product<GU, 1, 32>(a, wc, xc, st);
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
    launch<false>(a, w->codes_dev, codes_dev, (cudaStream_t)stream);
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
    launch<true>(a, w->codes_dev, codes_dev, (cudaStream_t)stream);
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
