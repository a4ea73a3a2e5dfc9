// Products of 8-bit rows in expert order with their experts' 8-bit matrices (include/moe_layer.h: moe_i8_product_device, moe_i8_gate_up_device) on the
// tensor core's integer product: the sums are exact, the scales of the row and of the matrix's row come last.
//
// A work item is 128 rows of one expert's matrix for each CTA that works on it (for gate_up 64 features, the gate row and the up row of each next to
// one another) times up to NT of the expert's rows. The matrix is the instruction's M side and the rows its N side, so a few rows cost a
// short instruction and what an item costs is bringing the matrix. Persistent units (a CTA, or a pair of CTAs on two SMs that share the rows:
// tcgen05's cta_group::2) take items in turn; items of one expert are neighbours.
//
// What bounds it: few rows an expert (1,000 over 512 experts of 2,048 x 512, of which 440 have some) HBM, 139 us of gate_up at 6.7 TB/s and 73 of the product at
// 6.3; many (65,536 over 128 of 2,560 x 768) what an SM takes in, 52 to 57 bytes a clock: a pair's stage brings each CTA 16 KB of the matrix and 64 bytes a
// row, which at 256 rows is 64 bytes for every clock of its MMAs, and more at fewer rows. 217 and 134 us (2.4 and 1.9 PTOP/s; HBM alone would take 118 and
// 97) at the 1.6 GHz that the tensor load leaves, 250 and 155 to 165 under a second of load; with two experts, whose matrices stay in the L2, 164 and 110. Without
// stores 214 and 112, without an epilogue 203 and 103; one large 8,192 x 8,192 x 8,192 370, 335 without (3.3 PTOP/s). Tried, and not faster: results through shared
// memory, by 16-byte stores or bulk-tensor copies; items of two pieces of the matrix, which bring a quarter less but leave no second accumulator (the large
// one 339, gate_up 228); stages of 256 values for pairs; 32 rows from tensor memory at a time. One row, 6.8 and 4.9 us, is latency.
//
// Roles of a CTA's warps: one thread brings the bytes by bulk-tensor copies, a stage of the contraction at a time; one lane (of a pair's first CTA)
// issues the MMAs; groups of four warps turn accumulators, of which there are two sets, into results.
//
// Every wait on an mbarrier is bounded: one that runs out raises the CTA's abort flag, the other waits return at once, and the CTA frees its tensor
// memory and counts itself among the device's CTAs that gave up (moe_ops_status) before it exits.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "i8_mma.cuh"
#include "mx4.cuh"
#include "ops_common.h"
#include "tensor_map.h"
#include "two.cuh"

namespace moe {
namespace {

constexpr uint32_t kMaxExperts = 512;
constexpr uint32_t kRowsM = 128;        // matrix rows a CTA takes
constexpr uint32_t kTileTable = 1024;   // tiles whose expert is looked up in a table
constexpr uint32_t kChunk = 16;         // rows an epilogue warp turns at a time
constexpr uint32_t kItemRing = 16;

// min(g, limit) and u held to +-limit. NaN passes through.
__device__ __forceinline__ void hold(Two &g, Two &u, float limit) {
  float a = g.lo(), b = g.hi(), c = u.lo(), d = u.hi();
  asm("min.NaN.f32 %0, %0, %4;\n\tmin.NaN.f32 %1, %1, %4;\n\tmin.NaN.f32 %2, %2, %4;\n\tmax.NaN.f32 %2, %2, %5;\n\tmin.NaN.f32 %3, %3, %4;\n\tmax.NaN.f32 %3, %3, %5;"
      : "+f"(a), "+f"(b), "+f"(c), "+f"(d)
      : "f"(limit), "f"(-limit));
  g = Two(a, b), u = Two(c, d);
}
// silu(g) * u in the approximate forms, for g from kFarGate on: the exponential's argument, 116 there, rounds by 2^-18. Below, where 1 / (1 + e^-g) is e^g
// to f32 and may be too small for it, while u makes of it what the result's type holds: e^(g / 4) four times, the large factor first.
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ Two swiglu_near(const Two &g, const Two &u) {
  const Two p = g * Two(-1.4426950408889634f);
  float e0, e1, r0, r1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(p.lo()));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(p.hi()));
  const Two d = Two(e0, e1) + Two(1.0f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d.lo()));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(d.hi()));
  return g * Two(r0, r1) * u;
}
__device__ __forceinline__ float swiglu_far(float g, float u) {
  const float p = expf(0.25f * g);
  return u * p * p * g * p * p;
}
__device__ __forceinline__ Two swiglu_any(const Two &g, const Two &u) {
  const Two h = swiglu_near(g, u);
  return Two(g.lo() < kFarGate ? swiglu_far(g.lo(), u.lo()) : h.lo(), g.hi() < kFarGate ? swiglu_far(g.hi(), u.hi()) : h.hi());
}

struct I8Args {
  const float *ws, *xs;  // scales of the matrices' rows and of the rows
  const int32_t *offsets;
  uint32_t E, N, K, R;
  uint32_t items_per_tile;  // items that share a tile of rows
  float limit;
  void *y;
  uint32_t *gave_up;  // the device's count
};

// Maps over the bytes of the matrices and, in boxes of 16, 32, 64 and 128 rows, of the rows.
constexpr uint32_t kBoxes = 4;
__host__ __device__ constexpr uint32_t box_rows(uint32_t i) { return 16u << i; }
struct I8Maps {
  CUtensorMap w, x[kBoxes];
};

// A form of the kernel: what it makes (GU: h of swiglu(gate, up), else the products), CTAs a unit has, the most rows of a tile, and its groups of four epilogue warps. Its shared memory: stages
// of bytes; the scales of a tile's rows, an epilogue warp its own; barriers; the experts' first rows and first tiles; the tiles' experts.
template <bool GU, uint32_t CTAS, uint32_t NT, uint32_t G>
struct I8Form {
  static constexpr uint32_t kGroups = G;
  static constexpr uint32_t kThreads = 32 * (2 + 4 * kGroups);
  // A stage holds 128 values of the contraction, 128 bytes of a row, of single CTAs twice as many: half the hand-overs where a stage's MMAs are short (100 rows
  // over 512 experts 151 us of gate_up with 128, 145 with 256; pairs 165 with 128, 171 with 256 and half the stages).
  static constexpr uint32_t kParts = CTAS == 2 ? 1 : 2, kStageK = 128 * kParts;
  static constexpr uint32_t kPartBytes = (kRowsM + NT / CTAS) * 128;
  static constexpr uint32_t kStageBytes = kParts * kPartBytes;
  static constexpr uint32_t kStages = CTAS == 2 ? 6 : 5;
  static constexpr uint32_t kRowScales = kStages * kStageBytes;
  static constexpr uint32_t kWarpScales = NT / kGroups;  // of a warp
  static constexpr uint32_t kBarriers = kRowScales + 4 * kGroups * kWarpScales * 4;
  static constexpr uint32_t kTables = kBarriers + 320;
  static constexpr uint32_t kTileExperts = kTables + 2 * (kMaxExperts + 1) * 4 + 8;
  static constexpr uint32_t kTileRows = kTileExperts + 2 * kTileTable;
  static constexpr uint32_t kBytes = kTileRows + 2 * kMaxExperts + 1024;  // and room to align the base to 1024
  static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
  static_assert(2 * kThreads > kMaxExperts, "two experts a thread");
  static_assert(kThreads / 32 * 4 <= kBarriers - kRowScales, "a word a warp in the scales' room");
  static constexpr uint32_t kCols = 2 * NT;  // of tensor memory: two accumulators
  static_assert(kCols <= 512 && (kCols & (kCols - 1)) == 0 && kCols >= 32, "tensor memory");
  static_assert(NT % (kChunk * kGroups) == 0, "a group's chunks");
};

enum : uint32_t { kCopyWarp = 0, kMmaWarp = 1, kEpilogueWarp = 2 };

template <class Out, bool GU, uint32_t CTAS, uint32_t NT, uint32_t G>
__global__ void __launch_bounds__(I8Form<GU, CTAS, NT, G>::kThreads, 1) k_i8_product(const __grid_constant__ I8Args a, const __grid_constant__ I8Maps maps) {
  using namespace tc;
  using SM = I8Form<GU, CTAS, NT, G>;
  constexpr uint32_t S = SM::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;  // the same in every lane, and known to be
  const uint32_t rank = CTAS == 2 ? cluster_ctarank() : 0, unit = blockIdx.x / CTAS, nunits = gridDim.x / CTAS;
  uint64_t *bars = (uint64_t *)(smem + SM::kBarriers);
  // Barriers: stages full, empty; accumulators full, empty. Of a pair the first CTA's "full" of stages and "empty" of accumulators take both CTAs' arrivals.
  constexpr uint32_t kEmpty = S, kAccFull = 2 * S, kAccEmpty = kAccFull + 2, kBars = kAccEmpty + 2;
  static_assert(8 * kBars + 8 + 4 * kItemRing <= 320 && kItemRing > S, "the barriers' room; no more items are under way than stages");
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](uint32_t i) { return bar0 + 8 * i; };
  uint32_t *tmem_slot = (uint32_t *)(bars + kBars);
  volatile uint32_t *abort = tmem_slot + 1;
  volatile uint32_t *item_rows = abort + 1;  // rows of an instruction of the items under way, from the copies' thread to the MMAs' warp
  uint32_t *first_row = (uint32_t *)(smem + SM::kTables), *first_tile = first_row + kMaxExperts + 1;  // [E + 1] each
  uint16_t *tile_expert = (uint16_t *)(smem + SM::kTileExperts);
  uint16_t *tile_rows = (uint16_t *)(smem + SM::kTileRows);  // an expert's tiles' rows, but for its last
  // The warps' sums of tiles, before the scales come: where no copy writes, as one was seen to overtake ordinary reads that only a barrier stands behind.
  uint32_t *warp_part = (uint32_t *)(smem + SM::kRowScales);
  uint32_t *error = (uint32_t *)abort;     // the waits' error word: the flag itself

  if (tid == 0) {
    for (uint32_t s = 0; s < S; s++) mbar_init(bar(s), CTAS), mbar_init(bar(kEmpty + s), 1);
    for (uint32_t b = 0; b < 2; b++) mbar_init(bar(kAccFull + b), 1), mbar_init(bar(kAccEmpty + b), CTAS * 4 * SM::kGroups);
    *abort = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if constexpr (CTAS == 2) pair_arrive();
  // Tensor memory is taken when the kernels before are done, and the next may come when it is: a kernel that held it while it waits for another on the
  // same SM, which asks for it later, would wait for ever.
  wait_for_predecessors();
  if (warp == kMmaWarp) {
    if constexpr (CTAS == 2)
      tmem_alloc_pair(smem_u32(tmem_slot), SM::kCols);
    else
      tmem_alloc(smem_u32(tmem_slot), SM::kCols);
  }
  // The experts' first rows and first tiles, and the tiles' experts, two experts a thread. Offsets are held to 0 .. R, and to rise: each to the largest
  // before it, which is looked for where one does not.
  {
    const uint32_t e = 2 * tid;
    auto row_of = [&](uint32_t x) { return a.offsets ? min((uint32_t)max(a.offsets[x], 0), a.R) : x ? a.R : 0u; };
    uint32_t r0 = e <= a.E ? row_of(e) : 0, r1 = e < a.E ? row_of(e + 1) : r0, r2 = e + 1 < a.E ? row_of(e + 2) : r1;
    if (__syncthreads_or(r1 < r0 || r2 < r1)) {
      for (uint32_t x = 0; x < min(e, a.E); x++) r0 = max(r0, row_of(x));
      r1 = max(r0, r1), r2 = max(r1, r2);
    }
    dependents_may_launch();
    const uint32_t t0 = (r1 - r0 + NT - 1) / NT, t1 = (r2 - r1 + NT - 1) / NT;
    uint32_t sum = t0 + t1;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= (uint32_t)off) sum += o;
    }
    if (lane == 31) warp_part[warp] = sum;
    __syncthreads();
    sum += __reduce_add_sync(0xffffffffu, lane < warp ? warp_part[lane] : 0) - t0 - t1;
    if (e <= a.E) first_row[e] = r0, first_tile[e] = sum;
    if (e < a.E) first_row[e + 1] = r1, first_tile[e + 1] = sum + t0;
    // An expert's rows are shared out evenly among as few tiles as hold them: a short last tile would cost its matrix's bringing all the same. In steps of 32, its
    // last tile the rest: of up to 8 tiles, whose rows are 32 (tiles - 1) more than 256 (tiles - 1) at most short of full, none is empty, and of more all are full.
    auto even = [&](uint32_t rows, uint32_t tiles) { return CTAS == 2 && tiles ? ((rows + tiles - 1) / tiles + 31) & ~31u : NT; };
    if (e < a.E) tile_rows[e] = (uint16_t)even(r1 - r0, t0);
    if (e + 1 < a.E) tile_rows[e + 1] = (uint16_t)even(r2 - r1, t1);
    for (uint32_t t = sum; t < min(sum + t0 + t1, kTileTable); t++) tile_expert[t] = (uint16_t)(t < sum + t0 ? e : e + 1);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) pair_wait();  // the other CTA's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t M = a.items_per_tile, K = a.K, F = a.N / 2, KT = (K + SM::kStageK - 1) / SM::kStageK, ntiles = first_tile[a.E];
  auto expert_at = [&](uint32_t t) {  // the last expert whose first tile is at most t
    uint32_t lo = 0, hi = a.E;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (first_tile[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t lead0 = CTAS == 2 ? map_to_cta(bar0, 0) : bar0;  // the first CTA's barriers as this CTA names them
  auto lead = [&](uint32_t i) { return lead0 + 8 * i; };
  bool ok = true;

  // Item i is piece m = i % M of the matrix for tile t = i / M of the experts' tiles in order; a unit steps by nunits items.
  struct Item {
    uint32_t t, m;
  };
  const uint32_t step_t = nunits / M, step_m = nunits - step_t * M;
  const Item first{unit / M, unit % M};
  auto step = [&](Item &i) {
    i.t += step_t, i.m += step_m;
    if (i.m >= M) i.m -= M, i.t++;
  };
  // row0: the first of this CTA's matrix rows, or of its features.
  struct Tile {
    uint32_t expert, start, count, row0;
  };
  auto tile_at = [&](const Item &i) {
    const uint32_t e = i.t < kTileTable ? tile_expert[i.t] : expert_at(i.t);
    const uint32_t rows = tile_rows[e], start = first_row[e] + (i.t - first_tile[e]) * rows;
    return Tile{e, start, min(rows, first_row[e + 1] - start), (i.m * CTAS + rank) * (GU ? kRowsM / 2 : kRowsM)};
  };
  // The rows an instruction takes of a tile: rounded up to 16 for every CTA.
  auto rounded = [&](uint32_t count) { return (count + 16 * CTAS - 1) & ~(16 * CTAS - 1); };

  if (warp == kCopyWarp) {
    if (lane == 0) {
      uint32_t s = 0, phase = 1, item = 0;  // of the stage's "empty": the first round finds it so
      for (Item i = first; i.t < ntiles && ok; step(i), item++) {
        const Tile t = tile_at(i);
        // A CTA of a pair brings its half of the instruction's rows, by one copy or two. A copy may run past the tile's rows; what it brings then goes
        // into columns nobody reads.
        const uint32_t half = rounded(t.count) / CTAS, x_row = t.start + rank * half;
        const uint32_t b0 = 27 - __clz(half), rest = half - box_rows(b0), b1 = rest > 16 ? 28 - __clz(rest - 1) : 0;
        const uint32_t bytes = (kRowsM + box_rows(b0) + (rest ? box_rows(b1) : 0)) * 128;
        for (uint32_t it = 0; it < KT && ok; it++) {
          ok = mbar_wait(bar(kEmpty + s), phase, abort, error);
          if (!ok) break;
          uint32_t at = smem_u32(smem + s * SM::kStageBytes), x0 = it * SM::kStageK;
          const uint32_t parts = SM::kParts == 1 ? 1 : min(SM::kParts, (K - x0 + 127) / 128);
          if (it == 0 && rank == 0) item_rows[item % kItemRing] = rounded(t.count);
          if constexpr (CTAS == 2)
            mbar_arrive_expect_cluster(lead(s), parts * bytes);
          else
            mbar_arrive_expect(lead(s), parts * bytes);
          for (uint32_t part = 0; part < parts; part++, at += SM::kPartBytes, x0 += 128) {
            tma_load_matrix<CTAS>(at, &maps.w, x0, GU ? 2 * t.expert : t.row0 / 32, GU ? t.row0 / 16 : t.expert, lead(s));
            tma_load_byte_rows<CTAS>(at + kRowsM * 128, &maps.x[b0], x0, x_row, lead(s));
            if (rest) tma_load_byte_rows<CTAS>(at + (kRowsM + box_rows(b0)) * 128, &maps.x[b1], x0, x_row + box_rows(b0), lead(s));
          }
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
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint32_t leader = elect_leader();
      auto commit = [&](uint32_t i) {
        if constexpr (CTAS == 2)
          mma_commit_pair(leader, bar(i), 3);
        else
          mma_commit(leader, bar(i));
      };
      const uint32_t stage0 = smem_u32(smem) >> 4, last = (K - 1) % SM::kStageK / 32 + 1;  // steps of the last stage
      uint32_t s = 0, phase = 0, b = 0, acc_phase = 1, item = 0, idesc = 0;
      for (Item i = first; i.t < ntiles && ok; step(i), item++) {
        const uint32_t acc = tmem_base + b * NT;
        ok = mbar_wait_warp(bar(kAccEmpty + b), acc_phase, abort, error);
        for (uint32_t it = 0; it < KT && ok; it++) {
          ok = mbar_wait_warp(bar(s), phase, abort, error);
          if (!ok) break;
          if (it == 0) idesc = i8_instr_desc(item_rows[item % kItemRing], CTAS * kRowsM);
          tc_fence_after();
          const uint32_t stage = stage0 + s * (SM::kStageBytes >> 4), rows = stage + (kRowsM * 128 >> 4), steps = it == KT - 1 ? last : 4 * SM::kParts;
#pragma unroll
          for (uint32_t k = 0; k < 4 * SM::kParts; k++) {
            const uint32_t at = k / 4 * (SM::kPartBytes >> 4) + 2 * (k % 4);
            if (k < steps) mma_i8<CTAS>(leader, acc, stage + at, rows + at, idesc, (it | k) != 0);
          }
          commit(kEmpty + s);
          if (++s == S) s = 0, phase ^= 1;
        }
        if (!ok) break;
        commit(kAccFull + b);
        acc_phase ^= b, b ^= 1;
      }
    }
  } else {
    // Warp w reads tensor memory's lanes 32 (w % 4) ...; the groups take chunks of 16 rows in turn. Of a chunk a thread has, of four lanes eight apart, the sums of
    // four rows, two neighbours and two eight on. The four lanes are four neighbouring rows of the matrix, or gate and up of two neighbouring features, as the map
    // laid them: a thread's results of a row lie side by side, and eight threads' too.
    const uint32_t q = warp % 4, group = (warp - kEpilogueWarp) / 4, of_eight = lane / 4, pair = 2 * (lane % 4);
    constexpr uint32_t dc = SM::kGroups * kChunk, kMine = GU ? 2 : 4;  // features of a thread
    const uint32_t c0 = group * kChunk, width = GU ? F : a.N;
    float *row_scales = (float *)(smem + SM::kRowScales) + (4 * group + q) * SM::kWarpScales;
    // The scales of a tile's rows that the warp turns, chunk after chunk, and of the thread's four matrix rows: loaded while the tile before is turned.
    constexpr uint32_t kHeld = (SM::kWarpScales + 31) / 32;
    float held[kHeld], s[4];
    auto bring = [&](const Tile &t) {
#pragma unroll
      for (uint32_t k = 0; k < kHeld; k++) {
        const uint32_t j = 32 * k + lane, r = c0 + j / kChunk * dc + j % kChunk;
        held[k] = r < t.count ? a.xs[t.start + r] : 0.0f;
      }
      const uint32_t f = t.row0 + (GU ? 16 : 32) * q;  // features come 32 together
      const float *ws = a.ws + (uint64_t)t.expert * a.N + f + kMine * of_eight;
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) s[i] = f < width ? ws[GU ? i % 2 + i / 2 * F : i] : 0.0f;
    };
    uint32_t b = 0, phase = 0;
    Tile t{};
    if (first.t < ntiles) bring(t = tile_at(first));
    for (Item i = first; i.t < ntiles && ok;) {
      const Tile now = t;
      const uint32_t from = tmem_base + ((32 * q) << 16) + b * NT, f = now.row0 + (GU ? 16 : 32) * q;
      const Two w[4] = {Two(s[0]), Two(s[1]), Two(s[2]), Two(s[3])};
      __syncwarp();  // the scales of the tile before are read
#pragma unroll
      for (uint32_t k = 0; k < kHeld; k++)
        if (32 * k + lane < SM::kWarpScales) row_scales[32 * k + lane] = held[k];
      __syncwarp();
      step(i);
      if (i.t < ntiles) bring(t = tile_at(i));
      ok = mbar_wait_warp(bar(kAccFull + b), phase, abort, error);
      if (!ok) break;
      tc_fence_after();
      const float *sx = row_scales;
      auto load = [&](uint32_t c, uint32_t *v) { tmem_ld_16x16(from + c, v), tmem_ld_16x16(from + (16 << 16) + c, v + 8); };
      // A chunk's sums are on their way from tensor memory while the one before is turned.
      auto turn = [&](uint32_t c, const uint32_t *v, const float *sx) {
        const float2 a0 = *(const float2 *)(sx + pair), a1 = *(const float2 *)(sx + 8 + pair);
        const Two x[2] = {Two(a0.x, a0.y), Two(a1.x, a1.y)};
        // Lane j's two rows, neighbours or (half 1) those eight on: the sums, the rows' scales, the matrix's row's.
        auto scaled = [&](uint32_t j, uint32_t half) {
          const uint32_t at = 8 * (j / 2) + 4 * half + 2 * (j % 2);
          return Two((float)(int32_t)v[at], (float)(int32_t)v[at + 1]) * x[half] * w[j];
        };
        auto both = [](float a, float b) { return pack2(a, b, (const Out *)nullptr); };
        Two r[2][kMine];
#pragma unroll
        for (uint32_t half = 0; half < 2; half++) {
          if constexpr (GU) {
            r[half][0] = scaled(0, half), r[half][1] = scaled(1, half);
            Two u[2] = {scaled(2, half), scaled(3, half)};
            if (a.limit > 0.0f) hold(r[half][0], u[0], a.limit), hold(r[half][1], u[1], a.limit);
            const float low = fminf(fminf(r[half][0].lo(), r[half][0].hi()), fminf(r[half][1].lo(), r[half][1].hi()));
            if (low < kFarGate)  // a NaN gate does not count here, and stays one
              r[half][0] = swiglu_any(r[half][0], u[0]), r[half][1] = swiglu_any(r[half][1], u[1]);
            else
              r[half][0] = swiglu_near(r[half][0], u[0]), r[half][1] = swiglu_near(r[half][1], u[1]);
          } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) r[half][j] = scaled(j, half);
          }
        }
        Out *p = (Out *)a.y + (uint64_t)(now.start + c + pair) * width + f + kMine * of_eight;
        const uint32_t left = f < width && now.count > c + pair ? now.count - c - pair : 0;  // rows from the thread's first on
        auto store = [&](uint32_t row, uint32_t half, bool second) {
          if (row >= left) return;
          auto of = [&](uint32_t j) { return second ? r[half][j].hi() : r[half][j].lo(); };
          if constexpr (GU)
            *(uint32_t *)(p + (uint64_t)row * width) = both(of(0), of(1));
          else
            *(uint2 *)(p + (uint64_t)row * width) = make_uint2(both(of(0), of(1)), both(of(2), of(3)));
        };
        store(0, 0, false), store(1, 0, true), store(8, 1, false), store(9, 1, true);
      };
      // The accumulator is given back once the warp's last sums are here.
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CTAS == 2)
            mbar_arrive_cluster(lead(kAccEmpty + b));
          else
            mbar_arrive(lead(kAccEmpty + b));
        }
      };
      uint32_t v[16], u[16];
      if (c0 < now.count)
        load(c0, v);
      else
        release();
      for (uint32_t c = c0; c < now.count; c += 2 * dc, sx += 2 * kChunk) {
        tmem_ld_wait16(v);
        if (c + dc < now.count)
          load(c + dc, u);
        else
          release();
        turn(c, v, sx);
        if (c + dc >= now.count) break;
        tmem_ld_wait16(u);
        if (c + 2 * dc < now.count)
          load(c + 2 * dc, v);
        else
          release();
        turn(c + dc, u, sx + kChunk);
      }
      phase ^= b, b ^= 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort) atomicAdd(a.gave_up, 1u);
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

template <class Out, bool GU, uint32_t CTAS, uint32_t NT, uint32_t G>
void launch_product(const I8Args &args, const void *wc, const void *xc, cudaStream_t st) {
  using Form = I8Form<GU, CTAS, NT, G>;
  constexpr auto kernel = k_i8_product<Out, GU, CTAS, NT, G>;
  I8Args a = args;
  int device = 0;
  CUDA_OK(cudaGetDevice(&device));
  a.gave_up = gave_up_count(device);
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
  I8Maps maps;
  maps.w = GU ? make_gate_up_map(wc, a.K, all, a.E, kRowsM) : make_matrix_map(wc, a.K, all, a.E, kRowsM);
  for (uint32_t i = 0; i < kBoxes; i++)
    if (box_rows(i) <= NT / CTAS) maps.x[i] = make_byte_rows_map(xc, a.K, a.R, box_rows(i));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension, at[1].val.clusterDim = {CTAS, 1, 1};
  cfg.gridDim = dim3(CTAS * (unsigned)std::min<uint64_t>(most, units)), cfg.blockDim = dim3(Form::kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cfg.attrs = at, cfg.numAttrs = CTAS;  // a single CTA is no cluster
  CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a, maps));
}

// Tiles of 256 rows by pairs of CTAs where experts have more than 28 rows on average (many then have more than 32, two tiles of a single CTA) and there are 32 items
// for pairs at least and more than a round of them for single CTAs; else of 32 by single CTAs. The average is over all experts, as the host does not know
// which have rows. gate_up and down by single CTAs and by pairs, us from a graph: 512 experts of 2,048 x 512, 10,000 rows 174 + 90 and 175 + 92, 16,000 173 + 93 and
// 176 + 97, 24,000 204 + 126 and 179 + 105; 128 of 2,560 x 768, 2,000 rows 80 + 44 and 82 + 46, 3,200 84 + 45 and 83 + 46, skewed by a Zipf law of 1.1 86 + 48 and
// 83 + 47, 4,800 88 + 51 and 84 + 48. One matrix: 2,080 x 1,440, 200 rows (9 items for pairs) 5.9 and 8.5, 400 (18) 8.7 and 8.7, 777 (36) 11.5 and 9.0; 8,192 x
// 4,096, 64 rows (32, and 128 for single CTAs) 11.2 and 13.9, 128 rows (32, and 256) 16.9 and 14.6.
//
// Two groups of epilogue warps, as more warps' stores and waits stand in the way of the two that bring bytes and issue MMAs (pairs, 65,536 rows over 128 experts of 2,560 x
// 768: the product 134 us, 147 with four groups, 144 with one); four for gate_up by pairs where the contraction is too short for two to be done beside it
// (16,384 rows over 32 experts, n_in and features 256 and 128 9.3 us, 11.3 with two; 768 and 384 17.4 and 20.7; 1,280 and 768 33.1 and 34.8; 1,536 and 1,024 46.7 and
// 47.2; 2,048 and 1,536 85.6 and 85.1, 111 and 102 under load).
template <class Out, bool GU>
void launch(const I8Args &a, const void *wc, const void *xc, cudaStream_t st) {
  const uint64_t pieces = (a.N + 255) / 256, tiles = (uint64_t)a.R / 256 + 1, single = ((uint64_t)a.R + 31) / 32 * ((a.N + 127) / 128);
  if (a.R <= 28ull * a.E || pieces * tiles < 32 || single <= 148)
    launch_product<Out, GU, 1, 32, 2>(a, wc, xc, st);
  else if (GU && a.K <= 1536)
    launch_product<Out, GU, 2, 256, GU ? 4 : 2>(a, wc, xc, st);
  else
    launch_product<Out, GU, 2, 256, 2>(a, wc, xc, st);
}

I8Args arguments(const moe_i8_weights *w, const float *scales, uint32_t R, const int32_t *offsets) {
  need(w != nullptr, "weights are required");
  need(w->n_experts >= 1 && w->n_experts <= kMaxExperts, "n_experts must be 1 .. 512");
  need(w->n_out >= 32 && w->n_out % 32 == 0 && w->n_out <= kMxMaxValues, "n_out must be a multiple of 32, 32 .. 65536");
  need(w->n_in >= 32 && w->n_in % 32 == 0 && w->n_in <= kMxMaxValues, "n_in must be a multiple of 32, 32 .. 65536");
  need(w->reserved == 0, "reserved must be 0");
  need(offsets || w->n_experts == 1, "offsets are required for more than one expert");
  need(R <= 1u << 24, "R must be at most 2^24");
  I8Args a{};
  a.ws = w->scales_dev, a.xs = scales;
  a.offsets = offsets, a.E = w->n_experts, a.N = w->n_out, a.K = w->n_in, a.R = R;
  return a;
}

template <bool GU>
void call(const I8Args &a, const moe_i8_weights *w, const void *codes, uint32_t type, cudaStream_t st) {
  need_device({{w->codes_dev, "weight codes", 16}, {a.ws, "weight scales", 4}, {codes, "codes", 16}, {a.xs, "scales", 4}, {a.offsets, "offsets", 4, true},
               {a.y, GU ? "h" : "y", 16}});
  if (type == MOE_TYPE_BF16)
    launch<__nv_bfloat16, GU>(a, w->codes_dev, codes, st);
  else
    launch<__half, GU>(a, w->codes_dev, codes, st);
}

}  // namespace

}  // namespace moe

using namespace moe;

extern "C" {

MOE_API moe_status moe_i8_product_device(const moe_i8_weights *w, const void *codes_dev, const float *scales_dev, uint32_t R, const int32_t *offsets_dev, void *y_dev,
                                         uint32_t y_type, void *stream) {
  return ops_call([&] {
    need(y_type == MOE_TYPE_F16 || y_type == MOE_TYPE_BF16, "y_type must be MOE_TYPE_F16 or MOE_TYPE_BF16");
    I8Args a = arguments(w, scales_dev, R, offsets_dev);
    if (R == 0) return;
    a.y = y_dev;
    call<false>(a, w, codes_dev, y_type, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_i8_gate_up_device(const moe_i8_weights *w, const void *codes_dev, const float *scales_dev, uint32_t R, const int32_t *offsets_dev,
                                         float swiglu_limit, void *h_dev, uint32_t h_type, void *stream) {
  return ops_call([&] {
    need(h_type == MOE_TYPE_F16 || h_type == MOE_TYPE_BF16, "h_type must be MOE_TYPE_F16 or MOE_TYPE_BF16");
    need(!(swiglu_limit < 0.0f) && swiglu_limit - swiglu_limit == 0.0f, "swiglu_limit must be 0 or a positive number");
    I8Args a = arguments(w, scales_dev, R, offsets_dev);
    need(a.N % 64 == 0, "gate and up rows together must be a multiple of 64");
    if (R == 0) return;
    a.y = h_dev, a.limit = swiglu_limit;
    call<true>(a, w, codes_dev, h_type, (cudaStream_t)stream);
  });
}

}  // extern "C"
