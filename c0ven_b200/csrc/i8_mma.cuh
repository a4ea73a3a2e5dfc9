// The tensor core's product of 8-bit integers (tcgen05.mma kind::i8): A and B signed bytes in shared memory, K-major with the 128-byte swizzle, 32
// values of the contraction an instruction (32 bytes of a row), 32-bit sums in tensor memory. A single CTA's N is a multiple of 16, a pair's of 32.
#pragma once

#include <cstdint>

#include "expert_tiles.cuh"

namespace moe {
namespace tc {

// kind::i8 instruction descriptor: A and B signed, sums s32 that wrap, M m, N n.
__device__ __forceinline__ uint32_t i8_instr_desc(uint32_t n, uint32_t m) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }
// D[tmem] (+)= A[128 rows] * B[n rows]^T over 32 values. CTAS 2: by a pair's first CTA, 128 rows of A and half of B's n rows in each CTA's
// shared memory.
template <uint32_t CTAS>
__device__ __forceinline__ void mma_i8(uint32_t leader, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
// A box of the map's tensor of bytes (tensor_map.h, make_bytes_map): 128 bytes from byte x (a multiple of 16) of the rows from y on, every part's of a
// row one after another, of matrix z. CTAS 2: by a CTA of a pair, into its own shared memory, the bytes counted on a barrier that may be the other CTA's.
template <uint32_t CTAS>
__device__ __forceinline__ void tma_load_bytes(uint32_t dst_smem, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(0), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(0), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// cluster_sync in two halves: what a thread wrote before the first is seen by the pair's threads after the second.
__device__ __forceinline__ void pair_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

}  // namespace tc
}  // namespace moe
