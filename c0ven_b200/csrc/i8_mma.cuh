// The tensor core's product of 8-bit integers (tcgen05.mma kind::i8): A and B signed bytes in shared memory, K-major with the 128-byte swizzle, 32
// values of the contraction an instruction (32 bytes of a row), 32-bit sums in tensor memory. A single CTA's N is a multiple of 16, a pair's of 32.
#pragma once

#include <cstdint>

#include "expert_tiles.cuh"

namespace moe {
namespace tc {

// kind::i8 instruction descriptor: A and B signed, sums s32 that wrap, M m, N n.
__device__ __forceinline__ uint32_t i8_instr_desc(uint32_t n, uint32_t m) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }
// The high word of both operands' descriptors: rows of 128 contiguous bytes whose 16-byte pieces are swizzled by the row's low three bits, eight rows 1,024 bytes on.
// The low word is the address / 16.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
// D[tmem] (+)= A[128 rows] * B[n rows]^T over 32 values at a, b / 16. CTAS 2: by a pair's first CTA, 128 rows of A and half of B's n rows in each CTA's shared memory.
template <uint32_t CTAS>
__device__ __forceinline__ void mma_i8(uint32_t leader, uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
        : "memory");
}
// Boxes of the maps' tensors of bytes (tensor_map.h), 128 bytes from byte x (a multiple of 16) of every row: of a matrix from places y and z of the map's last two
// dimensions on (make_matrix_map, make_gate_up_map); of rows those from y on (make_byte_rows_map). CTAS 2: by a CTA of a pair, into its own shared memory, the bytes counted
// on a barrier that may be the other CTA's.
template <uint32_t CTAS>
__device__ __forceinline__ void tma_load_matrix(uint32_t dst_smem, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(0), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %4, %5}], [%6];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(0), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
template <uint32_t CTAS>
__device__ __forceinline__ void tma_load_byte_rows(uint32_t dst_smem, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// Sixteen lanes by sixteen columns of tensor memory: thread i has of lane i / 4 columns 2 (i % 4) and the next, in v[0] and v[1], of lane i / 4 + 8 the same in v[2] and
// v[3], and of columns 8 on in v[4] .. v[7].
__device__ __forceinline__ void tmem_ld_16x16(uint32_t taddr, uint32_t *v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr)
               : "memory");
}
// cluster_sync in two halves: what a thread wrote before the first is seen by the pair's threads after the second.
__device__ __forceinline__ void pair_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

}  // namespace tc
}  // namespace moe
