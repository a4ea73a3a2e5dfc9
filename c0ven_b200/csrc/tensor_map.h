// Tensor maps for the bulk-tensor (TMA) copies of the tile kernels' activation rows.
#pragma once

#include <cuda.h>

#include <cstdint>

namespace moe {

constexpr uint32_t kMapBoxRows = 64;  // rows one copy brings: a tile of n rows takes ceil(n / 64) copies a stage

// A map over f16 rows [rows][K] in device memory (base 16-byte aligned, K a multiple of 64) whose copies bring a box of
// 64 values x 64 rows into shared memory with the 128-byte swizzle, the layout the tensor core reads K-major operands
// in. Rows past `rows` read as zero. Throws CudaFailure when the driver refuses the map.
// box_rows: the rows one copy brings, at most 256 (the tensor must be at least that high).
CUtensorMap make_rows_map(const void *base, uint64_t rows, uint32_t K, uint32_t box_rows = kMapBoxRows);

// A map over the quants run of a weight matrix in the runs layout, for types whose rows' quants are one run of
// row_bytes bytes a row (Q4_K: K / 2): bytes [rows][row_bytes] per expert slot, the slots slice_bytes apart. A copy
// brings box_bytes of 128 rows of one slot, swizzled by box_bytes (64 or 128), so that the decode warps' 16-byte reads
// of neighbouring rows fall on different banks.
CUtensorMap make_quants_map(const void *base, uint32_t row_bytes, uint32_t rows, uint32_t nslots, uint64_t slice_bytes, uint32_t box_bytes);

// A map over matrices of 4-bit codes two a byte, [matrices][parts][rows][row_bytes] one after another (base 16-byte aligned, row_bytes a
// multiple of 16), whose copies bring 128 bytes (256 values) of box_rows rows of every part of one matrix, part after part, with the 128-byte
// swizzle. What lies past a row's end or past a part's rows reads as zero.
CUtensorMap make_codes_map(const void *base, uint32_t row_bytes, uint32_t rows, uint32_t parts, uint32_t matrices, uint32_t box_rows);

// Maps over matrices of bytes, [matrices][rows][row_bytes] one after another (base 16-byte aligned, row_bytes a multiple of 16, rows of 32), whose copies bring 128
// bytes of box_rows rows (a multiple of 32) of one matrix with the 128-byte swizzle. Every 32 of them come in the order 0, 4, ... 28, 1, 5, ... 29, 2, ... 30, 3, ... 31: a
// thread that has four lanes eight apart of a product has four neighbouring rows of the matrix. Places: of 32 rows, of matrices.
CUtensorMap make_matrix_map(const void *base, uint32_t row_bytes, uint32_t rows, uint32_t matrices, uint32_t box_rows);
// The same of matrices of rows gate and then rows up rows, whose copies bring box_rows / 2 of each: 0, 2, ... 14, 1, 3, ... 15 of 16 gate rows, then the same of 16 up
// rows, and so on. Places: of gate and of up matrices (matrix m's gate is 2 m), of 16 rows.
CUtensorMap make_gate_up_map(const void *base, uint32_t row_bytes, uint32_t rows, uint32_t matrices, uint32_t box_rows);

// A map over rows of bytes [rows][row_bytes] (base 16-byte aligned, row_bytes a multiple of 16), whose copies bring 128 bytes of box_rows rows with the 128-byte
// swizzle; zeros past the end.
CUtensorMap make_byte_rows_map(const void *base, uint32_t row_bytes, uint32_t rows, uint32_t box_rows);

}  // namespace moe
