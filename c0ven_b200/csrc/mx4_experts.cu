// Products of MX rows in expert order with their experts' MX matrices (include/moe_layer.h: moe_mx4_product_device, moe_mx4_gate_up_device),
// on the tensor core's own 4-bit product: nothing is decoded.
//
// A work item is 128 rows of one expert's matrix for each CTA that works on it (for gate_up 64 gate rows and the 64 up rows of the same
// features) times up to NT of the expert's rows. The matrix is the instruction's M side and the rows its N side, so a few rows cost a
// short instruction and what an item costs is bringing the matrix. Persistent units (a CTA, or a pair of CTAs on two SMs that share the rows:
// tcgen05's cta_group::2) take items in turn; items of one expert are neighbours.
//
// What bounds it: few rows an expert (1,000 over 512 experts of 2,048 x 512) HBM, 75 us of gate_up at 6.5 TB/s and 43 of the product at 5.8; many
// (65,536 over 128 of 2,560 x 768) no one unit, 150 and 106 us at 3.4 and 2.4 PFLOP/s (5.3 on a dense 8,192 x 8,192 x 8,192). Taken apart in an earlier
// build on another GPU, where the whole took 148 and 104: 123 and 66 without the epilogues, 104 and 57 without scales too. One row, 7.4 and 5 us, is
// latency: 1,300 cycles until the experts' first rows are here, 700 for the tables, 2,600 until the first scales are in tensor memory, 490 a stage of
// MMAs, 1,500 from the last to the end.
//
// Roles of a CTA's warps: one thread brings codes by bulk-tensor copies, 256 values of the contraction a stage; three warps bring the scales,
// four stages (1,024 values: a sector of a row's scales) at a time in turn, word by word into the layout that the tensor core's copy reads
// (an expert's first row lies anywhere, so rows' scales cannot be laid out in advance; the matrices', which could, have the same form); one lane (of a pair's first CTA) issues the copies of
// scales to tensor memory, and one the MMAs; groups of four warps turn accumulators, of which there are two sets, into results.
//
// Every wait on an mbarrier is bounded: one that runs out raises the CTA's abort flag, the other waits return at once, and the CTA frees its tensor
// memory and counts itself among the device's CTAs that gave up (moe_ops_status) before it exits.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <type_traits>
#include <utility>

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
constexpr uint32_t kTileTable = 1024;   // tiles whose expert is looked up in a table
constexpr uint32_t kChunk = 16;         // rows an epilogue warp turns at a time
constexpr uint32_t kPiece = 528;        // bytes from a piece of 512 bytes of scales to the next: the eight words of a row fall on different banks

// Barriers of two epilogue warps alone. The second tells both whether ok holds for both: they leave their loop together or not at all, so
// that neither waits here for one that has left.
__device__ __forceinline__ void two_warps_sync(uint32_t id) { asm volatile("bar.sync %0, 64;" ::"r"(1 + id) : "memory"); }
__device__ __forceinline__ bool two_warps_all(uint32_t id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(1 + id)
      : "memory");
  return r != 0;
}

// Eight lanes hold eight 4-bit codes each, code j of lane i becomes code i of lane j: three exchanges of the half a lane does not keep, by halves,
// by bytes and by codes.
struct CodeTranspose {
  uint32_t halves, bytes, shift, keep;
  __device__ explicit CodeTranspose(uint32_t lane)
      : halves(lane & 4 ? 0x3276u : 0x5410u), bytes(lane & 2 ? 0x3715u : 0x6240u), shift(lane & 1 ? 28 : 4), keep(lane & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu) {}
  __device__ uint32_t operator()(uint32_t v) const {
    v = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 4), halves);
    v = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 2), bytes);
    const uint32_t c = __shfl_xor_sync(0xffffffffu, v, 1);
    return (v & keep) | (__funnelshift_l(c, c, shift) & ~keep);
  }
};

// min(g, limit) and u held to +-limit. NaN passes through.
__device__ __forceinline__ void hold(float &g, float &u, float limit) {
  asm("min.NaN.f32 %0, %0, %2;\n\tmin.NaN.f32 %1, %1, %2;\n\tmax.NaN.f32 %1, %1, %3;" : "+f"(g), "+f"(u) : "f"(limit), "f"(-limit));
}
// silu(g) * u in the approximate forms: two significant bits of it stay. For g from kFarGate on; the exponential's argument, 116 there, rounds by
// 2^-18.
__device__ __forceinline__ float swiglu_mx(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
}
// Below, where 1 / (1 + e^-g) is e^g to f32 and may be too small for it, while u makes of it what a scale can hold: e^(g / 4) four times, the large
// factor first. (Looking for such gates and the code for them cost 65,536 rows over 128 experts of 2,560 x 768 2 us of 148, a single row 0.6 of 6.9; the code as
// a function that is called 4.)
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ float swiglu_far(float g, float u) {
  const float p = expf(0.25f * g);
  return u * p * p * g * p * p;
}
// The warp's largest magnitude; NaN if there is one.
__device__ __forceinline__ float largest_magnitude(float v) {
  float m;
  asm("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

__device__ uint32_t g_gave_up;  // CTAs that gave up a wait, ever: whoever asks compares it with what they were told last
__global__ void k_note_give_up() { atomicAdd(&g_gave_up, 1u); }

struct Mx4Args {
  const uint8_t *ws, *xs;   // scales of the matrices and the rows
  const int32_t *offsets;
  uint32_t E, N, K, R;
  uint32_t items_per_tile;  // items that share a tile of rows
  float limit;
  void *y;
  uint8_t *hc, *hs;
};

// Maps over the codes of the matrices and, in boxes of 16, 32, 64 and 104 rows, of the rows.
constexpr uint32_t kBoxes = 4;
__host__ __device__ constexpr uint32_t box_rows(uint32_t i) { return i == 3 ? 104u : 16u << i; }
struct Mx4Maps {
  CUtensorMap w, x[kBoxes];
};

// What a form of the kernel makes: h as MX rows of swiglu(gate, up), or the products in Y.
struct GateUp {};

// A form of the kernel: what it makes, CTAs a unit has, and the most rows of a tile. Its shared memory: stages of codes; slots of scales, the matrix's
// and then the rows', eight words of every row each; for gate_up the accumulators that two warps exchange, twice 1 KB a warp; barriers; the experts' first rows and first tiles; the tiles' experts.
template <class Out, uint32_t CTAS, uint32_t NT>
struct Mx4Form {
  static constexpr bool GU = std::is_same<Out, GateUp>::value;
  static constexpr uint32_t kGroups = CTAS == 1 ? 1 : GU ? 4 : 2;  // of four epilogue warps
  static constexpr uint32_t kThreads = 32 * (6 + 4 * kGroups);
  static constexpr uint32_t kStages = CTAS == 2 ? 5 : 6;
  static constexpr uint32_t kStageBytes = (kRowsM + NT / CTAS) * 128;
  static constexpr uint32_t kScaleSlots = 3;  // and as many warps to fill them
  // A word of 128 rows' scales is a piece of 512 bytes and four columns of tensor memory, even where there are fewer rows: an instruction's scales
  // begin at a multiple of four columns.
  static constexpr uint32_t kRowPieces = (NT + 127) / 128;
  static constexpr uint32_t kScales = kStages * kStageBytes;
  static constexpr uint32_t kSlotBytes = 8 * (1 + kRowPieces) * kPiece;
  static constexpr uint32_t kStaging = kScales + kScaleSlots * kSlotBytes;
  static constexpr uint32_t kBarriers = kStaging + (GU ? 4 * kGroups * 2048 : 0);
  static constexpr uint32_t kTables = kBarriers + 320;
  static constexpr uint32_t kTileExperts = kTables + 2 * (kMaxExperts + 1) * 4;
  static constexpr uint32_t kBytes = kTileExperts + 2 * kTileTable + 1024;  // and room to align the base to 1024
  static_assert(kBytes <= 227 * 1024, "a CTA's shared memory");
  static_assert(2 * kThreads > kMaxExperts, "two experts a thread");
  static_assert(kThreads <= 32 * 32, "a lane a warp");
  // Tensor memory: two accumulators, then sets of columns for scales, of kScaleStages stages where they have the room, else of one. From the MMAs of
  // a unit of stages to those that find its columns filled again takes three hand-overs between warps, longer than the MMAs of a stage: with two
  // sets of one stage, beside accumulators of 224 columns, every stage waited 0.14 us.
  static constexpr uint32_t kStageCols = 2 * 4 * (1 + kRowPieces);
  static constexpr uint32_t kUnitStages = 2 * NT + 3 * kScaleStages * kStageCols <= 512 ? kScaleStages : 1;
  static constexpr uint32_t kSets = kUnitStages == 1 ? 4 : 3;
  // A stage is full when the CTAs' codes are there and, where units are single stages, its scales in tensor memory: one wait of the MMAs' warp less
  // (3 % of a dense gate_up of 8,192 x 8,192 x 8,192).
  static constexpr uint32_t kStageArrivals = CTAS + (kUnitStages == 1 ? 1 : 0);
  static constexpr uint32_t kUnitCols = kUnitStages * kStageCols;
  static constexpr uint32_t kUsedCols = 2 * NT + kSets * kUnitCols;
  static constexpr uint32_t kCols = kUsedCols <= 256 ? 256 : 512;
  static_assert(kUsedCols <= kCols, "tensor memory");
  static_assert(kSets < kStages, "the stage whose MMAs a set waits for has not been filled again");
};

enum : uint32_t { kCopyWarp = 0, kMmaWarp = 1, kScaleWarp = 2, kScaleCopyWarp = 5, kEpilogueWarp = 6 };

template <class Out, uint32_t CTAS, uint32_t NT>
__global__ void __launch_bounds__(Mx4Form<Out, CTAS, NT>::kThreads, 1) k_mx4_product(const __grid_constant__ Mx4Args a, const __grid_constant__ Mx4Maps maps) {
  using namespace tc;
  using SM = Mx4Form<Out, CTAS, NT>;
  constexpr bool GU = SM::GU;
  constexpr uint32_t S = SM::kStages, SL = SM::kScaleSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = CTAS == 2 ? cluster_ctarank() : 0, unit = blockIdx.x / CTAS, nunits = gridDim.x / CTAS;
  uint64_t *bars = (uint64_t *)(smem + SM::kBarriers);
  // Barriers: stages full, empty; scales full, empty; accumulators full, empty; sets of scales in tensor memory full, empty
  // (where a unit is a stage, the stage's own say that). Of a pair the first CTA's "full" of stages and scales and "empty"
  // of accumulators take both CTAs' arrivals.
  constexpr uint32_t kEmpty = S, kScFull = 2 * S, kScEmpty = kScFull + SL, kAccFull = kScEmpty + SL, kAccEmpty = kAccFull + 2, kSetFull = kAccEmpty + 2,
                     kSetEmpty = kSetFull + SM::kSets, kBars = kSetEmpty + SM::kSets;
  static_assert(8 * kBars + 8 <= 320, "the barriers' room");
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](uint32_t i) { return bar0 + 8 * i; };
  uint32_t *tmem_slot = (uint32_t *)(bars + kBars);
  volatile uint32_t *abort = tmem_slot + 1;
  uint32_t *first_row = (uint32_t *)(smem + SM::kTables), *first_tile = first_row + kMaxExperts + 1;  // [E + 1] each
  uint16_t *tile_expert = (uint16_t *)(smem + SM::kTileExperts);
  uint32_t *warp_part = (uint32_t *)(smem + SM::kScales);  // before the scales come
  uint32_t *error = (uint32_t *)abort;  // the waits' error word: the flag itself

  if (tid == 0) {
    for (uint32_t s = 0; s < S; s++) mbar_init(bar(s), SM::kStageArrivals), mbar_init(bar(kEmpty + s), 1);
    for (uint32_t s = 0; s < SL; s++) mbar_init(bar(kScFull + s), CTAS), mbar_init(bar(kScEmpty + s), 1);
    for (uint32_t b = 0; b < 2; b++) mbar_init(bar(kAccFull + b), 1), mbar_init(bar(kAccEmpty + b), CTAS * 4 * SM::kGroups);
    for (uint32_t b = 0; b < SM::kSets; b++) mbar_init(bar(kSetFull + b), 1), mbar_init(bar(kSetEmpty + b), 1);
    *abort = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if constexpr (CTAS == 2) cluster_arrive();
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
    for (uint32_t t = sum; t < min(sum + t0 + t1, kTileTable); t++) tile_expert[t] = (uint16_t)(t < sum + t0 ? e : e + 1);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_wait();  // the other CTA's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t M = a.items_per_tile, K = a.K, F = a.N / 2, KT = (K + kStageK - 1) / kStageK, ntiles = first_tile[a.E];
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
  auto arrive_lead = [&](uint32_t i) {
    if constexpr (CTAS == 2)
      mbar_arrive_cluster(lead(i));
    else
      mbar_arrive(lead(i));
  };
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
    const uint32_t start = first_row[e] + (i.t - first_tile[e]) * NT;
    return Tile{e, start, min(NT, first_row[e + 1] - start), (i.m * CTAS + rank) * (GU ? kRowsM / 2 : kRowsM)};
  };

  if (warp == kCopyWarp) {
    if (lane == 0) {
      uint32_t s = 0, phase = 1;  // of the stage's "empty": the first round finds it so
      for (Item i = first; i.t < ntiles && ok; step(i)) {
        const Tile t = tile_at(i);
        // A CTA of a pair brings its half of the rows the instruction takes, which are rounded up to 16: by one copy, or two. A copy may run past
        // the tile's rows; what it brings then goes into columns nobody reads. (Copies of 16 rows, seven a stage for a full tile, took 260 us
        // of a step whose copies take 141 so.)
        const uint32_t half = ((t.count + 15) & ~15u) / CTAS, x_row = t.start + rank * half;
        const uint32_t b0 = half > 80 ? 3 : half > 48 ? 2 : half > 16 ? 1 : 0, rest = half > box_rows(b0) ? box_rows(0) : 0;
        const uint32_t bytes = (kRowsM + box_rows(b0) + rest) * 128;
        for (uint32_t it = 0; it < KT && ok; it++) {
          ok = mbar_wait(bar(kEmpty + s), phase, abort, error);
          if (!ok) break;
          const uint32_t at = smem_u32(smem + s * SM::kStageBytes), x0 = it * (kStageK / 2);
          if constexpr (CTAS == 2)
            mbar_arrive_expect_cluster(lead(s), bytes);
          else
            mbar_arrive_expect(lead(s), bytes);
          tma_load_codes<CTAS>(at, &maps.w, x0, t.row0, t.expert, lead(s));
          tma_load_codes<CTAS>(at + kRowsM * 128, &maps.x[b0], x0, x_row, 0, lead(s));
          if (rest) tma_load_codes<CTAS>(at + (kRowsM + box_rows(b0)) * 128, &maps.x[0], x0, x_row + box_rows(b0), 0, lead(s));
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
    // A slot of scales by a warp, a word a lane: eight words of rows i, i + 32, i + 64 and i + 96 an instruction, so that a row's 32 bytes are one
    // request; the words, at 16 i + 4 (row / 32) of pieces 528 bytes apart, fall on 32 banks. Where the rest of a row is four words or fewer, those of
    // rows i + 4, ... too. (With loads into registers, 16 on their way at once, gate_up of 65,536 rows took 386 us where this took 182: what counts is
    // that a slot's copies are all on their way.) Only the bytes behind a row's last in its word are made zeros, as codes are there: words behind it are
    // not copied on, and rows behind the tile's or the matrix's go into results nobody reads.
    const uint32_t mine = warp - kScaleWarp, srow = mx_scale_row_bytes(K), nb = K / kMxBlock, slots = (KT + kScaleStages - 1) / kScaleStages;
    const uint32_t at = smem_u32(smem + SM::kScales + mine * SM::kSlotBytes);
    uint32_t turn = 0, phase = 1;  // whose turn the next slot is
    for (Item i = first; i.t < ntiles && ok; step(i)) {
      const Tile t = tile_at(i);
      for (uint32_t j = 0; j < slots && ok; j++, turn = turn == SL - 1 ? 0 : turn + 1) {
        if (turn != mine) continue;
        ok = mbar_wait_warp(bar(kScEmpty + mine), phase, abort, error);
        if (!ok) break;
        phase ^= 1;
        // The lane's word, and its first row of each 128. Its bytes of a row's scales: n from b0 on.
        constexpr uint32_t kSlotBlocks = kScaleStages * kStageK / kMxBlock;
        const bool few = nb - j * kSlotBlocks <= kSlotBlocks / 2;
        const uint32_t word = lane % (few ? 4 : 8), quarter = few ? lane / 4 % 4 : lane / 8, r0 = few ? lane / 16 * 4 : 0, every = few ? 8 : 4;
        const uint32_t b0 = j * kSlotBlocks + 4 * word, n = b0 < nb ? min(4u, nb - b0) : 0u;
        const uint32_t to = at + word * kPiece + 4 * quarter + 16 * r0;
        // Rows src + 0 .. 3, every + 0 .. 3, ... of 32, have of them, to the places from `to` on.
        auto bring = [&](uint32_t to, const uint8_t *src, uint32_t have) {
          const uint64_t skip = (uint64_t)(every - 4) * srow;
          if (__all_sync(0xffffffffu, have >= 32 - r0 && (n == 4 || n == 0))) {
            if (n)
#pragma unroll 2
              for (uint32_t k = 0; k < 32; k += every, to += 16 * every, src += skip)
#pragma unroll
                for (uint32_t u = 0; u < 4; u++, src += srow) copy_word(to + 16 * u, src);
            return;
          }
          for (uint32_t k = 0; k < 32; k += every, to += 16 * every, src += skip)
#pragma unroll
            for (uint32_t u = 0; u < 4; u++, src += srow)
              if (n && k + u < have) copy_word(to + 16 * u, src, n);
        };
        {
          const uint32_t r = 32 * quarter + r0, row = GU ? (r < 64 ? t.row0 + r : F + t.row0 + r - 64) : t.row0 + r;
          bring(to, a.ws + ((uint64_t)t.expert * a.N + row) * srow + b0, row < a.N ? a.N - row : 0);
        }
        if constexpr (NT <= 32) {
          // Up to 32 rows, which lie in the first column of a piece: neighbours an instruction.
          const uint32_t lanes = few ? 4 : 8;
          if (n)
            for (uint32_t r = lane / lanes; r < t.count; r += 32 / lanes) copy_word(at + (8 + word) * kPiece + 16 * r, a.xs + (uint64_t)(t.start + r) * srow + b0, n);
        } else {
          for (uint32_t p = 0; p < SM::kRowPieces && 128 * p < t.count; p++) {
            const uint32_t r = 128 * p + 32 * quarter + r0;
            bring(to + 8 * (1 + p) * kPiece, a.xs + (uint64_t)(t.start + r) * srow + b0, r < t.count ? t.count - r : 0);
          }
        }
        copy_words_wait();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive_lead(kScFull + mine);
      }
    }
  } else if (warp == kScaleCopyWarp) {
    // Scales to tensor memory, a unit of stages at a time, while the MMAs of the unit before run: an MMA waits for every copy that the same thread
    // issued before it, which cost a stage of a full tile a third of its time.
    if (rank == 0) {
      constexpr uint32_t U = SM::kUnitStages;
      const uint32_t leader = elect_leader();
      // The MMAs of kSets units ago, which read the set's columns, are done: a unit of one stage has that stage's "empty" say so.
      uint32_t stage = 0, slot = 0, slot_phase = 0, set = 0, done = U == 1 ? S - SM::kSets : 0, done_phase = 1;
      for (Item i = first; i.t < ntiles && ok; step(i)) {
        for (uint32_t it = 0; it < KT && ok; it += U) {
          const uint32_t sub = it % kScaleStages;
          if (sub == 0) ok = mbar_wait_warp(bar(kScFull + slot), slot_phase, abort, error);
          if (ok) ok = mbar_wait_warp(bar((U == 1 ? kEmpty : kSetEmpty) + done), done_phase, abort, error);
          if (!ok) break;
          if (++done == (U == 1 ? S : SM::kSets)) done = 0, done_phase ^= 1;
          tc_fence_after();
          const uint32_t to = tmem_base + 2 * NT + set * SM::kUnitCols, to_rows = to + 8 * U, from = smem_u32(smem + SM::kScales + slot * SM::kSlotBytes);
          const uint32_t words = min(2 * U, (K - it * kStageK + 127) / 128);
#pragma unroll
          for (uint32_t w = 0; w < 2 * U; w++) {
            if (w >= words) continue;
            copy_scales<CTAS>(leader, to + 4 * w, from + (2 * sub + w) * kPiece);
#pragma unroll
            for (uint32_t p = 0; p < SM::kRowPieces; p++)
              copy_scales<CTAS>(leader, to_rows + 4 * (w * SM::kRowPieces + p), from + (8 * (1 + p) + 2 * sub + w) * kPiece);
          }
          const uint32_t full = bar(U == 1 ? stage : kSetFull + set);
          if constexpr (CTAS == 2)
            mma_commit_pair(leader, full, 1);
          else
            mma_commit(leader, full);
          if (++stage == S) stage = 0;
          if (sub + U == kScaleStages || it + U >= KT) {
            if constexpr (CTAS == 2)
              mma_commit_pair(leader, bar(kScEmpty + slot), 3);
            else
              mma_commit(leader, bar(kScEmpty + slot));
            if (++slot == SL) slot = 0, slot_phase ^= 1;
          }
          if (++set == SM::kSets) set = 0;
        }
      }
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      constexpr uint32_t U = SM::kUnitStages;
      const uint32_t leader = elect_leader();
      auto commit = [&](uint32_t i, uint32_t ctas) {
        if constexpr (CTAS == 2)
          mma_commit_pair(leader, bar(i), ctas);
        else
          mma_commit(leader, bar(i));
      };
      uint32_t s = 0, phase = 0, set = 0, set_phase = 0, b = 0, acc_phase = 1;
      for (Item i = first; i.t < ntiles && ok; step(i)) {
        const Tile t = tile_at(i);
        const uint32_t n = (t.count + 15) & ~15u, acc = tmem_base + b * NT;
        const uint32_t d0 = mx4_instr_desc(n, CTAS * kRowsM, 0), d2 = mx4_instr_desc(n, CTAS * kRowsM, 2);
        ok = mbar_wait_warp(bar(kAccEmpty + b), acc_phase, abort, error);
        for (uint32_t it = 0; it < KT && ok; it++) {
          const uint32_t in_unit = it % U, ta = tmem_base + 2 * NT + set * SM::kUnitCols, tb = ta + 8 * U;
          if (U > 1 && in_unit == 0) ok = mbar_wait_warp(bar(kSetFull + set), set_phase, abort, error);
          if (ok) ok = mbar_wait_warp(bar(s), phase, abort, error);
          if (!ok) break;
          tc_fence_after();
          const uint32_t stage = smem_u32(smem + s * SM::kStageBytes), rows = stage + kRowsM * 128;
          const uint32_t steps = min(4u, (K - it * kStageK + 63) / 64);
#pragma unroll
          for (uint32_t k = 0; k < 4; k++) {
            const uint32_t w = 2 * in_unit + k / 2;
            if (k < steps)
              mma_mx4<CTAS>(leader, acc, smem_desc_sw128(stage + 32 * k), smem_desc_sw128(rows + 32 * k), k % 2 ? d2 : d0, ta + 4 * w,
                            tb + 4 * SM::kRowPieces * w, (it | k) != 0);
          }
          commit(kEmpty + s, 3);
          if (++s == S) s = 0, phase ^= 1;
          if (in_unit == U - 1 || it == KT - 1) {
            if constexpr (U > 1) commit(kSetEmpty + set, 1);
            if (++set == SM::kSets) set = 0, set_phase ^= 1;
          }
        }
        if (!ok) break;
        commit(kAccFull + b, 3);
        acc_phase ^= b, b ^= 1;
      }
    }
  } else if (warp >= kEpilogueWarp) {
    // Warp w reads tensor memory's lanes 32 (w % 4) ...; the groups take chunks of 16 rows in turn.
    const uint32_t q = warp % 4, group = (warp - kEpilogueWarp) / 4;
    uint32_t b = 0, phase = 0;
    [[maybe_unused]] const CodeTranspose transpose(lane);
    for (Item i = first; i.t < ntiles && ok; step(i)) {
      const Tile t = tile_at(i);
      const uint32_t from = tmem_base + ((32 * q) << 16) + b * NT;
      ok = mbar_wait_warp(bar(kAccFull + b), phase, abort, error);
      if constexpr (GU) ok = two_warps_all(2 * group + q % 2, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t c0 = group * kChunk, dc = SM::kGroups * kChunk;
      if constexpr (!GU) {
        // A lane holds one feature of 16 rows. Two lanes with neighbouring features share out two rows: the even one stores both features of the
        // first, the odd one of the second. A chunk's values are on their way from tensor memory while the one before is stored.
        const uint32_t odd = lane & 1, sel = odd ? 0x3276u : 0x5410u;
        auto store = [&](uint32_t c, const uint32_t *v) {
          Out *p = (Out *)a.y + (uint64_t)(t.start + c + odd) * a.N + (t.row0 + 32 * q + lane - odd);
          const uint32_t left = t.count - c;
#pragma unroll
          for (uint32_t j = 0; j < 16; j += 2, p += 2 * a.N) {
            const uint32_t mine = pack2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), (const Out *)nullptr), theirs = __shfl_xor_sync(0xffffffffu, mine, 1);
            if (j + odd < left) *(uint32_t *)p = __byte_perm(mine, theirs, sel);
          }
        };
        if (t.row0 + 32 * q < a.N) {  // features come 32 together
          uint32_t v[16], u[16];
          if (c0 < t.count) tmem_ld16(from + c0, v);
          for (uint32_t c = c0; c < t.count; c += 2 * dc) {
            tmem_ld_wait16(v);
            if (c + dc < t.count) tmem_ld16(from + c + dc, u);
            store(c, v);
            if (c + dc >= t.count) break;
            tmem_ld_wait16(u);
            if (c + 2 * dc < t.count) tmem_ld16(from + c + 2 * dc, v);
            store(c + dc, u);
          }
        }
      } else {
        // Warps q and q + 2 hold gate and up of the same 32 features, a lane's one feature of 16 rows. They exchange: the first takes both of the
        // chunk's first eight rows, the other of its last eight. A block of h is then a row's 32 lanes. The exchange has two places, by turns:
        // when one is written again both warps have passed the barrier that came after its reading.
        const uint32_t up = q / 2, at = t.row0 + 32 * (q % 2), hrow = mx_scale_row_bytes(F);
        float *mine = (float *)(smem + SM::kStaging) + (4 * group + q) * 512 + lane, *theirs = (float *)(smem + SM::kStaging) + (4 * group + (q ^ 2)) * 512 + lane;
        const uint32_t keep_at = from + 8 * up, give_at = from + 8 - 8 * up;
        uint32_t r = c0 + 8 * up + lane % 8;  // the row whose codes this lane gets
        uint8_t *hc = a.hc + (uint64_t)(t.start + r) * (F / 2) + at / 2 + 4 * (lane / 8), *hs = a.hs + (uint64_t)(t.start + r) * hrow + at / kMxBlock;
        uint32_t keep[8], give[8], turn = 0;
        if (c0 < t.count) tmem_ld8(keep_at + c0, keep), tmem_ld8(give_at + c0, give);
        for (uint32_t c = c0; c < t.count; c += dc, r += dc, hc += (uint64_t)dc * (F / 2), hs += (uint64_t)dc * hrow, turn ^= 256) {
          tmem_ld_wait8(keep), tmem_ld_wait8(give);
          float h[8];
#pragma unroll
          for (uint32_t j = 0; j < 8; j++) mine[turn + 32 * j] = __uint_as_float(give[j]), h[j] = __uint_as_float(keep[j]);
          if (c + dc < t.count) tmem_ld8(keep_at + c + dc, keep), tmem_ld8(give_at + c + dc, give);
          two_warps_sync(2 * group + q % 2);
          float got[8];
#pragma unroll
          for (uint32_t j = 0; j < 8; j++) got[j] = theirs[turn + 32 * j];
          auto make_h = [&](float (&g)[8], float (&u)[8]) {
            if (a.limit > 0.0f)
#pragma unroll
              for (uint32_t j = 0; j < 8; j++) hold(g[j], u[j], a.limit);
            float low = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) low = fminf(low, g[j]);
            if (low < kFarGate) {  // h may be g or u
#pragma unroll
              for (uint32_t j = 0; j < 8; j++) h[j] = g[j] < kFarGate ? swiglu_far(g[j], u[j]) : swiglu_mx(g[j], u[j]);
            } else {
#pragma unroll
              for (uint32_t j = 0; j < 8; j++) h[j] = swiglu_mx(g[j], u[j]);
            }
          };
          if (up)
            make_h(got, h);
          else
            make_h(h, got);
          // The rows' scales: f is the exponent of the largest magnitude, at least 2; 2^(127 - (f - 2)) is what the values are multiplied by. A lane works
          // one out, of row lane % 8, and the rows' eight lanes hand theirs round. A row with an infinity or NaN (f 255) gets codes 0.
          float top = 0.0f;
#pragma unroll
          for (uint32_t j = 0; j < 8; j++) {
            const float m = largest_magnitude(h[j]);
            if (lane % 8 == j) top = m;
          }
          const uint32_t f = max(__float_as_uint(top) & 0x7F800000u, 2u << 23);
#pragma unroll
          for (uint32_t j = 0; j < 8; j++) h[j] *= __uint_as_float(0x80000000u - __shfl_sync(0xffffffffu, f, j));
          // The warp's eight rows by eight features: lane j of each eight gets row j's codes of those features.
          uint32_t codes = transpose(mx_codes8(h));
          const bool bad = f == 0x7F800000u;
          if (bad) codes = 0;
          if (r < t.count && at < F) {
            *(uint32_t *)hc = codes;
            if (lane < 8) {
              *hs = bad ? 255 : (uint8_t)((f >> 23) - 2);
              if (at + kMxBlock == F)
                for (uint32_t z = 1; z < hrow - (F / kMxBlock - 1); z++) hs[z] = 0;
            }
          }
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
  if (tid == 0 && *abort) atomicAdd(&g_gave_up, 1u);
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

template <class Out, uint32_t CTAS, uint32_t NT>
void launch_product(const Mx4Args &args, const void *wc, const void *xc, cudaStream_t st) {
  using Form = Mx4Form<Out, CTAS, NT>;
  constexpr auto kernel = k_mx4_product<Out, CTAS, NT>;
  constexpr bool GU = Form::GU;
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
  Mx4Maps maps;
  maps.w = make_codes_map(wc, a.K / 2, all, GU ? 2 : 1, a.E, GU ? kRowsM / 2 : kRowsM);
  for (uint32_t i = 0; i < kBoxes; i++) maps.x[i] = make_codes_map(xc, a.K / 2, a.R, 1, 1, box_rows(i));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension, at[1].val.clusterDim = {CTAS, 1, 1};
  cfg.gridDim = dim3(CTAS * (unsigned)std::min<uint64_t>(most, units)), cfg.blockDim = dim3(Form::kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cfg.attrs = at, cfg.numAttrs = CTAS;  // a single CTA is no cluster
  CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a, maps));
}

// Tiles of 208 rows by pairs of CTAs where experts have more than 26 rows on average (many then have more than 32, two tiles of a single CTA) and there
// are 32 items for pairs at least; else of 32 by single CTAs. The average is over all experts, as the host does not know which have rows. gate_up and
// down by pairs and by single CTAs, us: 512 experts of 2,048 x 512, 10 rows 8.4 + 5.6 and 7.4 + 5.0, 1,000 rows 78 + 43 and 75 + 43, 12,000 rows 94 + 54
// and 92 + 53, 14,000 rows 95 + 55 and 94 + 57, 16,000 rows 95 + 56 and 104 + 68, 32,000 rows 99 + 65 and 177 + 125; 128 of 2,560 x 768, 2,800 rows 48 + 27
// and 46 + 26, skewed by a Zipf law of 1.1 47 + 28 and 52 + 30; one of 2,080 x 1,440, 200 rows (12 items for pairs) 11 + 8 and 10 + 6, 777 rows (48) 12 + 8
// and 16 + 10; one of 8,192 x 4,096, 128 rows (32) 15 + 10 and 23 + 13.
template <class Out>
void launch(const Mx4Args &a, const void *wc, const void *xc, cudaStream_t st) {
  const uint64_t pieces = (a.N + 255) / 256, tiles = (uint64_t)a.R / 208 + 1;
  if (a.R > 26ull * a.E && pieces * tiles >= 32)
    launch_product<Out, 2, 208>(a, wc, xc, st);
  else
    launch_product<Out, 1, 32>(a, wc, xc, st);
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
    a.y = y_dev;
    if (y_type == MOE_TYPE_BF16)
      launch<__nv_bfloat16>(a, w->codes_dev, codes_dev, (cudaStream_t)stream);
    else
      launch<__half>(a, w->codes_dev, codes_dev, (cudaStream_t)stream);
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
    launch<GateUp>(a, w->codes_dev, codes_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_ops_status(uint32_t timeout_ms, void *stream) {
  return ops_call([&] {
    cudaStream_t st = (cudaStream_t)stream;
    Stream::wait_on(st, timeout_ms);
    int device = 0;
    CUDA_OK(cudaGetDevice(&device));
    uint32_t gave_up = 0;
    CUDA_OK(cudaMemcpyFromSymbolAsync(&gave_up, g_gave_up, sizeof gave_up, 0, cudaMemcpyDeviceToHost, st));
    Stream::wait_on(st, timeout_ms);
    if (!gave_up) return;
    // What this thread was told about the stream last. Nothing is cleared: others hear of the same products.
    thread_local std::map<std::pair<int, cudaStream_t>, uint32_t> told;
    uint32_t &last = told[{device, st}];
    if (last == gave_up) return;
    last = gave_up;
    throw Timeout("a product gave up waiting for its copies or its products: the results of products since this thread last asked are not to be used");
  });
}

MOE_API moe_status moe_ops_note_give_up(void *stream) {
  return ops_call([&] { CUDA_OK(launch_kernel(false, k_note_give_up, dim3(1), dim3(1), 0, (cudaStream_t)stream)); });
}

}  // extern "C"
