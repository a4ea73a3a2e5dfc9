// Rows to and from microscaled 4-bit floating point, and the combine without a layer. All are single passes over their data: what bounds rows to and
// from MX, and the combine of rows of 512 values and more, is HBM (figures at each).
#include <cuda_runtime.h>

#include <cstdint>

#include "mx4.cuh"
#include "ops_common.h"

namespace moe {
namespace {

constexpr uint32_t kRowsMaxUsed = 16;

// How rows are dealt to a CTA of 256 threads: 2^log2 neighbouring threads a row, eight values each (grid.y where a row has more), and U rows a
// thread, whose loads are on their way together. Four rows a thread where that leaves every SM some four CTAs: 32,768 rows of 2,048 bf16
// values to MX rows and back take 32 + 27 us so (5.3 and 6.2 TB/s) and 43 + 37 with one, bound by the loads' round trip and the CTAs' coming and
// going; f32 values to MX rows 44 us, 6.8 TB/s. 13 rows of 2,560 to eight places each and back take 1.9 + 1.7 us, one round trip after another.
constexpr uint32_t kManyOctets = 4 * 148 * 4 * 256;
template <uint32_t U>
struct RowsMap {
  static constexpr uint32_t kRows = U;
  uint32_t T, log2;
  __device__ uint32_t octet() const { return (blockIdx.y << log2) + (threadIdx.x & ((1u << log2) - 1)); }
  __device__ uint64_t row(uint32_t u) const { return ((uint64_t)blockIdx.x * U + u) * (256u >> log2) + (threadIdx.x >> log2); }
};

// The largest magnitude's bits among eight values as f32's, an infinity's or NaN's if there is one: magnitudes order as their bits do, and 16-bit
// types' are compared two at a time.
__device__ __forceinline__ uint32_t largest_bits(const uint4 (&raw)[2], const float *) {
  const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, w[i] & 0x7FFFFFFFu);
  return m;
}
__device__ __forceinline__ uint32_t largest_bits(const uint4 (&raw)[1], const __nv_bfloat16 *) {
  constexpr uint32_t kBits = 0x7FFF7FFFu;
  uint32_t p;
  asm("{\n\t.reg .b32 q;\n\tmax.NaN.bf16x2 %0, %1, %2;\n\tmax.NaN.bf16x2 q, %3, %4;\n\tmax.NaN.bf16x2 %0, %0, q;\n\t}"
      : "=&r"(p) : "r"(raw[0].x & kBits), "r"(raw[0].y & kBits), "r"(raw[0].z & kBits), "r"(raw[0].w & kBits));
  return max(p & 0x7FFF0000u, p << 16);
}
__device__ __forceinline__ uint32_t largest_bits(const uint4 (&raw)[1], const __half *) {
  constexpr uint32_t kBits = 0x7FFF7FFFu;
  uint32_t p;
  asm("{\n\t.reg .b32 q;\n\tmax.NaN.f16x2 %0, %1, %2;\n\tmax.NaN.f16x2 q, %3, %4;\n\tmax.NaN.f16x2 %0, %0, q;\n\t}"
      : "=&r"(p) : "r"(raw[0].x & kBits), "r"(raw[0].y & kBits), "r"(raw[0].z & kBits), "r"(raw[0].w & kBits));
  const float2 f = __half22float2(*(const __half2 *)&p);
  return max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu);
}

// Four threads hold a block of 32. Rows stay as they were loaded until their turn.
template <class X, uint32_t U>
__global__ void __launch_bounds__(256) k_mx4_quantize(const X *x, uint64_t stride, const RowsMap<U> map, uint32_t K, const int32_t *inv, uint32_t n_used, uint32_t R,
                                                      uint8_t *codes, uint8_t *scales) {
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t k = 8 * map.octet(), srow = mx_scale_row_bytes(K), b = k / kMxBlock;
  const bool in = k < K;  // K is a multiple of 32: a block's four threads alike
  uint4 raw[U][sizeof(X) / 2];
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t t = map.row(u);
#pragma unroll
    for (uint32_t i = 0; i < sizeof(X) / 2; i++) raw[u][i] = in && t < map.T ? ((const uint4 *)(x + t * stride + k))[i] : make_uint4(0, 0, 0, 0);
  }
  // All of the warp's lanes exchange before any is done: narrow rows are several a warp, and the last of them ends some lanes' work before others'.
  uint32_t top[U];
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    uint32_t m = largest_bits(raw[u], (const X *)nullptr);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    top[u] = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t t = map.row(u);
    if (t >= map.T) break;
    const uint32_t scale = mx_scale_of(top[u]);
    const float f = mx_inverse(scale);
    float v[8];
    load8((const X *)raw[u], v);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= f;
    const uint32_t c = scale == 255 ? 0u : mx_codes8(v);
    for (uint32_t j = 0; j < (inv ? n_used : 1); j++) {
      const uint64_t r = inv ? (uint64_t)(uint32_t)inv[t * n_used + j] : t;
      if (r >= R) continue;
      if (in) *(uint32_t *)(codes + r * (K / 2) + k / 2) = c;
      if (threadIdx.x % 4 == 0 && b < srow) scales[r * srow + b] = in ? (uint8_t)scale : 0;
    }
  }
}

template <class Y, uint32_t U>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, const RowsMap<U> map, uint32_t K, Y *out) {
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t k = 8 * map.octet(), srow = mx_scale_row_bytes(K);
  if (k >= K) return;
  uint32_t c[U], s[U];
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t r = map.row(u);
    c[u] = s[u] = 0;
    if (r < map.T) c[u] = *(const uint32_t *)(codes + r * (K / 2) + k / 2), s[u] = scales[r * srow + k / kMxBlock];
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t r = map.row(u);
    if (r >= map.T) break;
    float v[8];
    mx_values8(c[u], v);
    const float f = mx_scale(s[u]);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= f;
    store8(out + r * K + k, v);
  }
}

// A thread a block of the file: its bytes hold value j and value j + 16, the rows' hold neighbours. A CTA a row of up to 8,192 values, of which narrower ones
// leave threads idle, and single bytes loaded, as 17 bytes have no alignment: 2.9 TB/s of 65,536 rows of 2,880, 2.1 of 327,680 of 2,048, 0.07 of 70,001 of 64.
// A file is brought in once.
__global__ void __launch_bounds__(256) k_mx4_from_blocks(const uint8_t *blocks, uint32_t K, uint8_t *codes, uint8_t *scales) {
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t r = blockIdx.x;
  const uint32_t b = blockIdx.y * 256 + threadIdx.x, srow = mx_scale_row_bytes(K);
  if (b >= srow) return;
  if (b >= K / kMxBlock) {
    scales[r * srow + b] = 0;
    return;
  }
  const uint8_t *p = blocks + (r * (K / kMxBlock) + b) * 17;
  scales[r * srow + b] = p[0];
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const uint32_t lo = p[1 + i], hi = p[2 + i];
    w[i / 8] |= ((lo & 15u) | (hi & 15u) << 4) << (i / 2 % 4 * 8);
    w[2 + i / 8] |= (lo >> 4 | (hi >> 4) << 4) << (i / 2 % 4 * 8);
  }
  *(uint4 *)(codes + r * (K / 2) + b * 16) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A thread takes 8 columns of a row; the loads of four results are on their way before the first is added. A CTA takes 2,048 columns of a row, and narrower
// rows leave its threads idle. At equal bytes, ten results each: rows of 2,048 values 6.1 TB/s, 4,096 6.1, 2,560 6.0, 1,536 5.9, 512 5.6, 64 1.2, where CTAs'
// coming and going is what bounds it.
template <class Y>
__global__ void __launch_bounds__(256) k_combine_rows(const Y *y, uint32_t R, const int32_t *inv, const float *w, uint32_t n_used, uint32_t E,
                                                      const float *res, float *out) {
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t t = blockIdx.x;
  const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * 8;
  if (c >= E) return;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t j = 0; j < n_used; j++) {
    const uint32_t r = (uint32_t)inv[t * n_used + j];
    if (r >= R) continue;
    const float wj = w[t * n_used + j];
    float v[8];
    load8(y + (uint64_t)r * E + c, v);
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = fmaf(wj, v[i], acc[i]);
  }
  if (res) {
    float v[8];
    load8(res + t * E + c, v);
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] += v[i];
  }
  store8(out + t * E + c, acc);
}

// Grids of (rows, pieces of a row): rows up to 2^31 - 1.
dim3 rows_grid(uint32_t rows, uint32_t per_row) { return dim3(rows, (per_row + 255) / 256); }

// Calls f with the map for rows of so many groups of eight values, and its grid.
template <class F>
void with_rows_map(uint32_t T, uint32_t octets, F &&f) {
  uint32_t log2 = 2;
  while (log2 < 8 && (1u << log2) < octets) log2++;
  auto go = [&](auto map, uint32_t u) {
    const uint32_t rows = u * (256u >> log2);
    f(map, dim3((T + rows - 1) / rows, (octets + (1u << log2) - 1) >> log2));
  };
  if ((uint64_t)T * octets >= kManyOctets)
    go(RowsMap<4>{T, log2}, 4);
  else
    go(RowsMap<1>{T, log2}, 1);
}

// Launches for rows of one type.
template <class X>
void quantize(const void *x, uint64_t stride, uint32_t T, uint32_t K, const int32_t *inv, uint32_t n_used, uint32_t R, void *codes, void *scales, cudaStream_t st) {
  with_rows_map(T, mx_scale_row_bytes(K) * 4, [&](auto map, dim3 grid) {  // the scales' filling has its threads too
    CUDA_OK(launch_kernel(true, k_mx4_quantize<X, decltype(map)::kRows>, grid, dim3(256), 0, st, (const X *)x, stride, map, K, inv, n_used, R,
                          (uint8_t *)codes, (uint8_t *)scales));
  });
}
template <class Y>
void dequantize(const void *codes, const void *scales, uint32_t R, uint32_t K, void *out, cudaStream_t st) {
  with_rows_map(R, K / 8, [&](auto map, dim3 grid) {
    CUDA_OK(launch_kernel(true, k_mx4_dequantize<Y, decltype(map)::kRows>, grid, dim3(256), 0, st, (const uint8_t *)codes, (const uint8_t *)scales, map, K, (Y *)out));
  });
}

void need_mx_row(uint32_t K) { need(K >= kMxBlock && K % kMxBlock == 0 && K <= kMxMaxValues, "a row's values must be a multiple of 32, 32 .. 65536"); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API uint32_t moe_mx4_scale_row_bytes(uint32_t K) { return mx_scale_row_bytes(K); }

MOE_API moe_status moe_mx4_quantize_rows_device(const void *x_dev, uint32_t type, uint64_t stride, uint32_t T, uint32_t K, const int32_t *inv_dev,
                                                uint32_t n_used, uint32_t R, void *codes_dev, void *scales_dev, void *stream) {
  return ops_call([&] {
    const uint32_t size = row_type_bytes(type);
    need(size != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_mx_row(K);
    need(stride == 0 || (stride >= K && stride < 1ull << 32 && stride * size % 16 == 0), "stride must be 0, or K at least with rows 16-byte aligned");
    need(inv_dev ? n_used >= 1 && n_used <= kRowsMaxUsed : R == T, "n_used must be 1 .. 16 with inv, and R be T without");
    need(T < 1u << 31 && R < 1u << 31, "T and R must be below 2^31");
    if (T == 0 || R == 0) return;
    need_device({{x_dev, "x", 16}, {inv_dev, "inv", 4, true}, {codes_dev, "codes", 16}, {scales_dev, "scales", 4}});
    const auto call = type == MOE_TYPE_F32 ? quantize<float> : type == MOE_TYPE_F16 ? quantize<__half> : quantize<__nv_bfloat16>;
    call(x_dev, stride ? stride : K, T, K, inv_dev, n_used, R, codes_dev, scales_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_mx4_dequantize_rows_device(const void *codes_dev, const void *scales_dev, uint32_t R, uint32_t K, void *out_dev,
                                                  uint32_t type, void *stream) {
  return ops_call([&] {
    need(row_type_bytes(type) != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_mx_row(K);
    need(R < 1u << 31, "R must be below 2^31");
    if (R == 0) return;
    need_device({{codes_dev, "codes", 16}, {scales_dev, "scales", 4}, {out_dev, "out", 16}});
    const auto call = type == MOE_TYPE_F32 ? dequantize<float> : type == MOE_TYPE_F16 ? dequantize<__half> : dequantize<__nv_bfloat16>;
    call(codes_dev, scales_dev, R, K, out_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_mx4_from_blocks_device(const void *blocks_dev, uint32_t R, uint32_t K, void *codes_dev, void *scales_dev, void *stream) {
  return ops_call([&] {
    need_mx_row(K);
    need(R < 1u << 31, "R must be below 2^31");
    if (R == 0) return;
    need_device({{blocks_dev, "blocks", 1}, {codes_dev, "codes", 16}, {scales_dev, "scales", 4}});
    CUDA_OK(launch_kernel(true, k_mx4_from_blocks, rows_grid(R, mx_scale_row_bytes(K)), dim3(256), 0, (cudaStream_t)stream, (const uint8_t *)blocks_dev, K,
                          (uint8_t *)codes_dev, (uint8_t *)scales_dev));
  });
}

MOE_API moe_status moe_combine_rows_device(const void *y_dev, uint32_t y_type, uint32_t R, const int32_t *inv_dev, const float *w_dev, uint32_t T,
                                           uint32_t n_used, uint32_t n_embd, const float *residual_dev, float *out_dev, void *stream) {
  return ops_call([&] {
    need(row_type_bytes(y_type) != 0, "y_type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need(n_used >= 1 && n_used <= kRowsMaxUsed, "n_used must be 1 .. 16");
    need(n_embd >= 8 && n_embd % 8 == 0 && n_embd <= 1u << 24, "n_embd must be a multiple of 8, at most 2^24");
    need(T < 1u << 31 && R < 1u << 31, "T and R must be below 2^31");
    if (T == 0) return;
    // With R 0 no row of y is read: it may be null then.
    need_device({{y_dev, "y", 16, R == 0}, {inv_dev, "inv", 4}, {w_dev, "w", 4}, {residual_dev, "residual", 16, true}, {out_dev, "out", 16}});
    const dim3 grid = rows_grid(T, n_embd / 8), block(256);
    cudaStream_t st = (cudaStream_t)stream;
    if (y_type == MOE_TYPE_F32)
      CUDA_OK(launch_kernel(true, k_combine_rows<float>, grid, block, 0, st, (const float *)y_dev, R, inv_dev, w_dev, n_used, n_embd, residual_dev, out_dev));
    else if (y_type == MOE_TYPE_F16)
      CUDA_OK(launch_kernel(true, k_combine_rows<__half>, grid, block, 0, st, (const __half *)y_dev, R, inv_dev, w_dev, n_used, n_embd, residual_dev, out_dev));
    else
      CUDA_OK(launch_kernel(true, k_combine_rows<__nv_bfloat16>, grid, block, 0, st, (const __nv_bfloat16 *)y_dev, R, inv_dev, w_dev, n_used, n_embd, residual_dev,
                            out_dev));
  });
}

}  // extern "C"
