// The tensor core's block-scaled 4-bit product (tcgen05.mma kind::mxf4): A and B e2m1 codes in shared memory, K-major with the 128-byte
// swizzle, 64 values of the contraction an instruction (32 bytes of a row); their scales, a byte per 32 values, in tensor memory.
//
// Scales reach tensor memory by tcgen05.cp from shared memory, 512 bytes a copy: 128 rows' words of four scales (128 values). Row r's word
// lies at 16 (r % 32) + 4 (r / 32) of the piece, and lands in lane r % 32 (of every warp's quarter) of column r / 32. An instruction takes bytes
// 0, 1 or 2, 3 of the words, named by its descriptor's scale ids 0 or 2. Its scales' first columns are multiples of four: with another one it
// faults.
#pragma once

#include <cstdint>

#include "expert_tiles.cuh"

namespace moe {
namespace tc {

// cluster_sync in two halves: what a thread wrote before the first is seen by the pair's threads after the second.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 32 rows of 16 bytes, no swizzle: 8 rows 128 bytes on.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
// CTAS 2: by a pair's first CTA, each CTA's scales from its own shared memory to its own tensor memory.
template <uint32_t CTAS>
__device__ __forceinline__ void copy_scales(uint32_t leader, uint32_t taddr, uint32_t smem_addr) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
        "l"(smem_desc_scales(smem_addr)), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr),
        "l"(smem_desc_scales(smem_addr)), "r"(leader)
        : "memory");
}
// kind::mxf4 instruction descriptor: A and B e2m1, e8m0 scales, M m, N n, both operands' scale ids id (0 or 2).
__device__ __forceinline__ uint32_t mx4_instr_desc(uint32_t n, uint32_t m, uint32_t id) {
  return (id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) | (id << 29);
}
// D[tmem] (+)= A[128 rows] * B[n rows]^T over 64 values. CTAS 2: by a pair's first CTA, 128 rows of A and half of B's n rows in each CTA's
// shared memory; each CTA's tensor memory holds its rows' scales of A and all of B's.
template <uint32_t CTAS>
__device__ __forceinline__ void mma_mx4(uint32_t leader, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scales_a, uint32_t scales_b,
                                        uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scales_a), "r"(scales_b), "r"(accumulate), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "setp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scales_a), "r"(scales_b), "r"(accumulate), "r"(leader)
        : "memory");
}
// A box of the map's tensor of codes (tensor_map.h, make_codes_map): 128 bytes from byte x (a multiple of 16) of the rows from y on, of all parts of
// matrix z. CTAS 2: by a CTA of a pair, into its own shared memory, the bytes counted on a barrier that may be the other CTA's.
template <uint32_t CTAS>
__device__ __forceinline__ void tma_load_codes(uint32_t dst_smem, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(y), "r"(0), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(y), "r"(0), "r"(z), "r"(bar)
                 : "memory");
}
// Four bytes into shared memory, the first n of them from memory and zeros behind (n 0: nothing is read).
__device__ __forceinline__ void copy_word(uint32_t dst, const void *src, uint32_t n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_word(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_words_wait() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

}  // namespace tc
}  // namespace moe
