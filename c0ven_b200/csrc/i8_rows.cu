// Rows to and from 8-bit integers with a scale each (include/moe_layer.h, "8-bit rows"). Single passes over their data.
#include <cuda_runtime.h>

#include <cstdint>

#include "mx4.cuh"
#include "ops_common.h"

namespace moe {
namespace {

constexpr uint32_t kRowsMaxUsed = 16;
constexpr uint32_t kThreads = 256;
constexpr uint32_t kHeldOctets = 8;  // groups of eight values a thread holds

// How rows are dealt to a CTA of 256 threads: 2^log2 neighbouring threads a row; of its octets, groups of eight values, thread i takes i,
// i + 2^log2 and so on, V at most.
struct RowsOfThreads {
  uint32_t T, log2, octets;
  __device__ uint32_t first() const { return threadIdx.x & ((1u << log2) - 1); }
  __device__ uint32_t octet(uint32_t v) const { return first() + (v << log2); }
};

template <class X>
struct Octet {
  uint4 raw[sizeof(X) / 2];
  __device__ void load(const X *p) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(X) / 2; i++) raw[i] = ((const uint4 *)p)[i];
  }
  __device__ void zero() {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(X) / 2; i++) raw[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ void values(float *v) const { load8((const X *)raw, v); }
  // The largest magnitude's bits as f32's: magnitudes order as their bits do, an infinity's or NaN's above all numbers'.
  __device__ uint32_t largest() const {
    float v[8];
    values(v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
  }
};

// A row's scale and what its values are multiplied by. bad: it holds an infinity or NaN.
struct RowScale {
  float top, scale, inverse;
  bool bad, small;
  __device__ explicit RowScale(uint32_t bits) {
    bad = bits >= 0x7F800000u;
    top = __uint_as_float(bits);
    scale = bad ? __uint_as_float(0x7FFFFFFFu) : __fdiv_rn(top, 127.0f);
    small = top < 1e-35f;  // 127 / top would pass f32's range, or x times it be less exact than codes take
    inverse = bad || top == 0.0f ? 0.0f : __fdiv_rn(127.0f, top);
  }
};

// Eight codes: rint(127 x / top) of exact numbers. x * inverse is within 127 * 2^-23 < 2^-16 of 127 x / top; where it lies nearer than 2^-15 to a border between
// two codes the quotient is taken in 64 bits. There 127 x is exact, and the quotient's rounding makes no border of what is none: a quotient of numbers of 31 and
// 24 bits that is not n + 1/2 is 2^-33 of itself away from it at least.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], const RowScale &s) {
  if (s.bad) return make_uint2(0, 0);
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: sums with it are whole numbers, in the low bits
  float q[8], far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float y = x[i] * s.inverse;
    q[i] = y + kMagic;
    far = fmaxf(far, fabsf(y - (q[i] - kMagic)));
  }
  if ((s.small && s.top != 0.0f) || far > 0.5f - 0x1p-15f) {
#pragma unroll 1
    for (int i = 0; i < 8; i++) {
      // Held in registers: no index that the compiler does not know.
      float v = x[0];
#pragma unroll
      for (int j = 1; j < 8; j++) v = i == j ? x[j] : v;
      const float c = (float)rint(127.0 * (double)v / (double)s.top) + kMagic;
#pragma unroll
      for (int j = 0; j < 8; j++) q[j] = i == j ? c : q[j];
    }
  }
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; i++) b[i] = __float_as_uint(q[i]);
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); };
  return make_uint2(four(b[0], b[1], b[2], b[3]), four(b[4], b[5], b[6], b[7]));
}

// The largest of a row's 2^log2 threads' values. The CTA's threads come here together.
__device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t log2, uint32_t *part) {
  for (uint32_t off = min(16u, (1u << log2) / 2); off; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (log2 > 5) {
    const uint32_t warp = threadIdx.x / 32, each = 1u << (log2 - 5);
    if (threadIdx.x % 32 == 0) part[warp] = m;
    __syncthreads();
    for (uint32_t i = 0; i < each; i++) m = max(m, part[(warp & ~(each - 1)) + i]);
  }
  return m;
}

// V octets a thread of each of U rows, whose loads are on their way together.
template <class X, uint32_t V, uint32_t U>
__global__ void __launch_bounds__(kThreads) k_i8_quantize(const X *x, uint64_t stride, const RowsOfThreads map, uint32_t K, const int32_t *inv, uint32_t n_used, uint32_t R,
                                                          uint8_t *codes, float *scales) {
  __shared__ uint32_t part[U][kThreads / 32];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t rows = kThreads >> map.log2;
  const uint64_t t0 = (uint64_t)blockIdx.x * U * rows + (threadIdx.x >> map.log2);
  Octet<X> o[U][V];
#pragma unroll
  for (uint32_t u = 0; u < U; u++)
#pragma unroll
    for (uint32_t v = 0; v < V; v++) {
      const uint64_t t = t0 + u * rows;
      if (t < map.T && map.octet(v) < map.octets)
        o[u][v].load(x + t * stride + 8 * map.octet(v));
      else
        o[u][v].zero();
    }
  uint32_t top[U];
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    top[u] = 0;
#pragma unroll
    for (uint32_t v = 0; v < V; v++) top[u] = max(top[u], o[u][v].largest());
    top[u] = row_max(top[u], map.log2, part[u]);
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t t = t0 + u * rows;
    if (t >= map.T) break;
    const RowScale s(top[u]);
    uint2 c[V];
#pragma unroll
    for (uint32_t v = 0; v < V; v++) {
      float f[8];
      o[u][v].values(f);
      c[v] = codes8(f, s);
    }
    for (uint32_t j = 0; j < (inv ? n_used : 1); j++) {
      const uint64_t r = inv ? (uint64_t)(uint32_t)inv[t * n_used + j] : t;
      if (r >= R) continue;
#pragma unroll
      for (uint32_t v = 0; v < V; v++)
        if (map.octet(v) < map.octets) *(uint2 *)(codes + r * K + 8 * map.octet(v)) = c[v];
      if (map.first() == 0) scales[r] = s.scale;
    }
  }
}

// Rows longer than threads hold, a CTA each: read twice, the second time from the L2.
template <class X>
__global__ void __launch_bounds__(kThreads) k_i8_quantize_long(const X *x, uint64_t stride, uint32_t K, const int32_t *inv, uint32_t n_used, uint32_t R, uint8_t *codes,
                                                               float *scales) {
  __shared__ uint32_t part[kThreads / 32];
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t t = blockIdx.x;
  const X *row = x + t * stride;
  uint32_t top = 0;
  for (uint32_t k = 8 * threadIdx.x; k < K; k += 8 * 4 * kThreads) {
    Octet<X> o[4];
#pragma unroll
    for (uint32_t v = 0; v < 4; v++) {
      if (k + 8 * v * kThreads < K)
        o[v].load(row + k + 8 * v * kThreads);
      else
        o[v].zero();
    }
#pragma unroll
    for (uint32_t v = 0; v < 4; v++) top = max(top, o[v].largest());
  }
  const RowScale s(row_max(top, 8, part));
  for (uint32_t k = 8 * threadIdx.x; k < K; k += 8 * kThreads) {
    Octet<X> o;
    o.load(row + k);
    float f[8];
    o.values(f);
    const uint2 c = codes8(f, s);
    for (uint32_t j = 0; j < (inv ? n_used : 1); j++) {
      const uint64_t r = inv ? (uint64_t)(uint32_t)inv[t * n_used + j] : t;
      if (r < R) *(uint2 *)(codes + r * K + k) = c;
    }
  }
  if (threadIdx.x < (inv ? n_used : 1)) {
    const uint64_t r = inv ? (uint64_t)(uint32_t)inv[t * n_used + threadIdx.x] : t;
    if (r < R) scales[r] = s.scale;
  }
}

template <class Y>
__global__ void __launch_bounds__(kThreads) k_i8_dequantize(const uint8_t *codes, const float *scales, const RowsOfThreads map, uint32_t K, Y *out) {
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t r = (uint64_t)blockIdx.x * (kThreads >> map.log2) + (threadIdx.x >> map.log2);
  if (r >= map.T) return;
  const float s = scales[r];
  for (uint32_t o = map.first(); o < map.octets; o += 1u << map.log2) {
    const uint2 c = *(const uint2 *)(codes + r * K + 8 * o);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)(int8_t)((i < 4 ? c.x : c.y) >> (8 * (i % 4))) * s;
    store8(out + r * K + 8 * o, v);
  }
}

uint32_t ceil_log2(uint32_t n) {
  uint32_t l = 0;
  while ((1u << l) < n) l++;
  return l;
}

template <class X>
void quantize(const void *x, uint64_t stride, uint32_t T, uint32_t K, const int32_t *inv, uint32_t n_used, uint32_t R, void *codes, void *scales, cudaStream_t st) {
  const uint32_t octets = K / 8;
  if (octets > kThreads * kHeldOctets) {
    CUDA_OK(launch_kernel(true, k_i8_quantize_long<X>, dim3(T), dim3(kThreads), 0, st, (const X *)x, stride, K, inv, n_used, R, (uint8_t *)codes, (float *)scales));
    return;
  }
  auto go = [&](auto v, auto u, uint32_t log2) {
    constexpr uint32_t V = decltype(v)::value, U = decltype(u)::value;
    const uint32_t rows = U * (kThreads >> log2);
    CUDA_OK(launch_kernel(true, k_i8_quantize<X, V, U>, dim3((T + rows - 1) / rows), dim3(kThreads), 0, st, (const X *)x, stride, RowsOfThreads{T, log2, octets}, K, inv,
                          n_used, R, (uint8_t *)codes, (float *)scales));
  };
  using std::integral_constant;
  const uint32_t log2 = std::min(8u, ceil_log2(octets)), held = (octets + (1u << log2) - 1) >> log2;
  if (held <= 1)
    go(integral_constant<uint32_t, 1>{}, integral_constant<uint32_t, 1>{}, log2);
  else if (held <= 2)
    go(integral_constant<uint32_t, 2>{}, integral_constant<uint32_t, 1>{}, log2);
  else if (held <= 4)
    go(integral_constant<uint32_t, 4>{}, integral_constant<uint32_t, 1>{}, log2);
  else
    go(integral_constant<uint32_t, 8>{}, integral_constant<uint32_t, 1>{}, log2);
}

template <class Y>
void dequantize(const void *codes, const void *scales, uint32_t R, uint32_t K, void *out, cudaStream_t st) {
  const uint32_t octets = K / 8, log2 = std::min(8u, ceil_log2(octets)), rows = kThreads >> log2;
  CUDA_OK(launch_kernel(true, k_i8_dequantize<Y>, dim3((R + rows - 1) / rows), dim3(kThreads), 0, st, (const uint8_t *)codes, (const float *)scales,
                        RowsOfThreads{R, log2, octets}, K, (Y *)out));
}

void need_i8_row(uint32_t K) { need(K >= 32 && K % 32 == 0 && K <= kMxMaxValues, "a row's values must be a multiple of 32, 32 .. 65536"); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API moe_status moe_i8_quantize_rows_device(const void *x_dev, uint32_t type, uint64_t stride, uint32_t T, uint32_t K, const int32_t *inv_dev,
                                               uint32_t n_used, uint32_t R, void *codes_dev, float *scales_dev, void *stream) {
  return ops_call([&] {
    const uint32_t size = row_type_bytes(type);
    need(size != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_i8_row(K);
    need(stride == 0 || (stride >= K && stride < 1ull << 32 && stride * size % 16 == 0), "stride must be 0, or K at least with rows 16-byte aligned");
    need(inv_dev ? n_used >= 1 && n_used <= kRowsMaxUsed : R == T, "n_used must be 1 .. 16 with inv, and R be T without");
    need(T < 1u << 31 && R < 1u << 31, "T and R must be below 2^31");
    if (T == 0 || R == 0) return;
    need_device({{x_dev, "x", 16}, {inv_dev, "inv", 4, true}, {codes_dev, "codes", 16}, {scales_dev, "scales", 4}});
    const auto call = type == MOE_TYPE_F32 ? quantize<float> : type == MOE_TYPE_F16 ? quantize<__half> : quantize<__nv_bfloat16>;
    call(x_dev, stride ? stride : K, T, K, inv_dev, n_used, R, codes_dev, scales_dev, (cudaStream_t)stream);
  });
}

MOE_API moe_status moe_i8_dequantize_rows_device(const void *codes_dev, const float *scales_dev, uint32_t R, uint32_t K, void *out_dev, uint32_t type,
                                                 void *stream) {
  return ops_call([&] {
    need(row_type_bytes(type) != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_i8_row(K);
    need(R < 1u << 31, "R must be below 2^31");
    if (R == 0) return;
    need_device({{codes_dev, "codes", 16}, {scales_dev, "scales", 4}, {out_dev, "out", 16}});
    const auto call = type == MOE_TYPE_F32 ? dequantize<float> : type == MOE_TYPE_F16 ? dequantize<__half> : dequantize<__nv_bfloat16>;
    call(codes_dev, scales_dev, R, K, out_dev, (cudaStream_t)stream);
  });
}

}  // extern "C"
