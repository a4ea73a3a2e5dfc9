// Rows to and from 8-bit integers with a scale each (include/moe_layer.h, "8-bit rows"). Single passes over their data: what bounds long calls is HBM. A row's values
// stay in its threads' registers, as they were loaded, from its largest magnitude to its codes. 32,768 rows of 2,048 bf16 values to 8-bit rows 35.5 us
// (5.7 TB/s) and back 31.5 (6.4); f32 values 58 (5.7); 65,536 rows of 768 bf16 values 30 (5.0), f32 49 (5.1); 300,000 of 64 bf16 15, f32 24.8; 4,096 of 2,880 bf16 to six
// places each 22, f32 31.7. 13 rows of 2,560 f32 values to eight places each and back 2.6 + 1.6 us, one round trip after another.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "mx4.cuh"
#include "ops_common.h"
#include "two.cuh"

namespace moe {
namespace {

constexpr uint32_t kRowsMaxUsed = 16;
constexpr uint32_t kThreads = 256;
constexpr uint32_t kHeldOctets = 8;             // groups of eight values a thread holds
// Octets of a call from which on a thread has up to eight of one row or more: as many as two CTAs an SM hold so. To 8-bit rows, us by an octet a thread and by up
// to eight: 2,048 bf16 values, 2,048 rows 5.7 and 5.6, 2,400 6.1 and 5.3, 4,800 11.0 and 7.2, 9,500 21 and 13.4; f32, 1,024 rows 4.2 and 4.6, 2,400 7.9 and 7.1, 9,500
// 31 and 21.5; 64 bf16 values, 75,800 rows 5.6 and 6.9, 152,000 9.3 and 8.9, 300,000 17.8 and 15.1. Back, by an octet a thread and by four: 2,400 rows of 2,048 3.4 and
// 3.8, 3,200 4.2 and 4.1, 9,500 12.6 and 10.7.
constexpr uint32_t kManyOctets = 2 * 148 * 256 * kHeldOctets;

// How rows are dealt to a CTA of 256 threads: 2^log2 neighbouring threads a row; of its octets, groups of eight values, thread i takes i,
// i + 2^log2 and so on.
struct RowsOfThreads {
  uint32_t T, log2, octets;
  __device__ uint32_t first() const { return threadIdx.x & ((1u << log2) - 1); }
  __device__ uint32_t octet(uint32_t v) const { return first() + (v << log2); }
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
  const uint32_t m = __vmaxu2(__vmaxu2(raw[0].x & kBits, raw[0].y & kBits), __vmaxu2(raw[0].z & kBits, raw[0].w & kBits));
  return max(m & 0x7FFF0000u, m << 16);
}
__device__ __forceinline__ uint32_t largest_bits(const uint4 (&raw)[1], const __half *) {
  constexpr uint32_t kBits = 0x7FFF7FFFu;
  const uint32_t m = __vmaxu2(__vmaxu2(raw[0].x & kBits, raw[0].y & kBits), __vmaxu2(raw[0].z & kBits, raw[0].w & kBits));
  const float2 f = __half22float2(*(const __half2 *)&m);
  return max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu);
}

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
  __device__ uint32_t largest() const { return largest_bits(raw, (const X *)nullptr); }
};

// A row's scale and what its values are multiplied by: 127 / top is inverse + rest to twice f32's digits. bad: it holds an infinity or NaN. lift: a power of two that
// takes the row away from the ends of f32's range, where 127 / top, products with 127 or what their roundings leave over would pass it; top, inverse and
// rest are the lifted row's.
struct RowScale {
  float top, scale, inverse, rest, lift;
  bool bad;
  RowScale() = default;
  __device__ explicit RowScale(uint32_t bits) {
    bad = bits >= 0x7F800000u;
    top = __uint_as_float(bits);
    scale = bad ? __uint_as_float(0x7FFFFFFFu) : __fdiv_rn(top, 127.0f);
    lift = top < 1e-30f && top != 0.0f ? 0x1p64f : top > 1e30f ? 0x1p-64f : 1.0f;
    top *= lift;
    inverse = bad || top == 0.0f ? 0.0f : __fdiv_rn(127.0f, top);
    rest = fmaf(-inverse, top, 127.0f) * (inverse * (1.0f / 127.0f));
  }
  __device__ bool odd() const { return bad || lift != 1.0f; }
};

// Eight codes: rint(127 x / top) of exact numbers, ties to even.
//
// Values of 16-bit types: the quotient is worked out to f32's nearest number y. A border between two codes, n + 1/2, is such a number; with x and top whole numbers
// below 2^11 times powers of two, a quotient in [2^e, 2^(e + 1)) that is not a border lies 2^(e - 20) from one at least, and y 2^(e - 23) from the quotient at most:
// y is a border where the quotient is, and on its side of it where it is not. (In rows whose largest has few bits one value in some 400 lies on a border.)
//
// f32 values: x * inverse, rounded once, is within 127 * 2^-23 < 2^-16 of 127 x / top. Where one lies nearer than 2^-15 to a border the sign of 127 x - border * top
// decides, from the two products and what their roundings left over: the products are near one another, so their difference is exact, and what was left
// over has ten bits at most. What a row lifted down loses of its smallest values is far below half a code.
//
// ODD: the row may be bad or lifted. (Looking for that at every eight values took 39 us where 35.5 do.)
template <class X, bool ODD>
__device__ __forceinline__ uint2 codes8(float (&x)[8], const RowScale &s) {
  if (ODD && s.bad) return make_uint2(0, 0);
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: sums with it are whole numbers, ties to even, in the low bits
  if (ODD && s.lift != 1.0f)
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] *= s.lift;
  const Two inverse(s.inverse), magic(kMagic);
  Two q[4];
  if constexpr (sizeof(X) == 2) {
    const Two rest(s.rest);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Two v(x[2 * i], x[2 * i + 1]);
      q[i] = fma(v, inverse, v * rest) + magic;
    }
  } else {
    const Two minus(-1.0f);
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Two v(x[2 * i], x[2 * i + 1]);
      q[i] = fma(v, inverse, magic);
      const Two off = fma(v, inverse, fma(q[i], minus, magic));
      most = fmaxf(most, fmaxf(fabsf(off.lo()), fabsf(off.hi())));
    }
    if (most > 0.5f - 0x1p-15f) {
      const Two n(127.0f), top(s.top);
      auto half = [](float v) { return copysignf(0.5f, v); };
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const Two v(x[2 * i], x[2 * i + 1]), code = q[i] + Two(-kMagic), off = fma(v, inverse, code * minus);
        const Two border = code + Two(half(off.lo()), half(off.hi())), a = n * v, b = (border * top) * minus;
        const Two over = (a + b) + fma(fma(border, top, b), minus, fma(n, v, a * minus));
        q[i] = (border + Two(over.lo() == 0.0f ? 0.0f : half(over.lo()), over.hi() == 0.0f ? 0.0f : half(over.hi()))) + magic;
      }
    }
  }
  auto four = [](const Two &a, const Two &b) {
    return __byte_perm(__byte_perm(__float_as_uint(a.lo()), __float_as_uint(a.hi()), 0x0040), __byte_perm(__float_as_uint(b.lo()), __float_as_uint(b.hi()), 0x0040), 0x5410);
  };
  return make_uint2(four(q[0], q[1]), four(q[2], q[3]));
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

// V octets a thread of each of U rows, whose loads are on their way together. CTAs an SM by the registers: five of 16-bit rows of one row a thread (35.5 us where four take
// 37.5), four where it has more (15 us of 300,000 rows of 64; five spill and take 17.7), two of f32 rows.
template <class X, uint32_t V, uint32_t U>
__global__ void __launch_bounds__(kThreads, sizeof(X) == 4 ? 2 : U == 1 ? 5 : 4) k_i8_quantize(const X *x, uint64_t stride, const RowsOfThreads map, uint32_t K, const int32_t *inv,
                                                                                              uint32_t n_used, uint32_t R, uint8_t *codes, float *scales) {
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
  RowScale s[U];
  bool odd = false;
#pragma unroll
  for (uint32_t u = 0; u < U; u++) s[u] = RowScale(top[u]), odd |= s[u].odd();
  auto write = [&](auto is_odd) {
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      const uint64_t t = t0 + u * rows;
      if (t >= map.T) break;
      const int32_t *to = inv + t * n_used;
#pragma unroll
      for (uint32_t v = 0; v < V; v++) {
        const uint32_t k = 8 * map.octet(v);
        float f[8];
        o[u][v].values(f);
        const uint2 c = codes8<X, decltype(is_odd)::value>(f, s[u]);
        if (k >= K) break;
        if (!inv)
          *(uint2 *)(codes + t * K + k) = c;
        else
          for (uint32_t j = 0; j < n_used; j++)
            if ((uint32_t)to[j] < R) *(uint2 *)(codes + (uint64_t)(uint32_t)to[j] * K + k) = c;
      }
      if (map.first() == 0) {
        if (!inv)
          scales[t] = s[u].scale;
        else
          for (uint32_t j = 0; j < n_used; j++)
            if ((uint32_t)to[j] < R) scales[(uint32_t)to[j]] = s[u].scale;
      }
    }
  };
  if (__any_sync(0xffffffffu, odd))
    write(std::true_type{});
  else
    write(std::false_type{});
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
    const uint2 c = codes8<X, true>(f, s);
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

// U rows' octets a thread, whose loads are on their way together.
template <class Y, uint32_t U>
__global__ void __launch_bounds__(kThreads) k_i8_dequantize(const uint8_t *codes, const float *scales, const RowsOfThreads map, uint32_t K, Y *out) {
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t rows = kThreads >> map.log2, k = 8 * ((blockIdx.y << map.log2) + map.first());
  const uint64_t r0 = (uint64_t)blockIdx.x * U * rows + (threadIdx.x >> map.log2);
  if (k >= K) return;
  uint2 c[U];
  float s[U];
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t r = r0 + u * rows;
    if (r < map.T) c[u] = *(const uint2 *)(codes + r * K + k), s[u] = scales[r];
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint64_t r = r0 + u * rows;
    if (r >= map.T) break;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)(int8_t)((i < 4 ? c[u].x : c[u].y) >> (8 * (i % 4))) * s[u];
    store8(out + r * K + k, v);
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
  // Long calls: up to eight octets a thread, of one row or more, by threads of one warp where a row has 2,048 values at most. Else an octet a thread where a CTA
  // has the threads.
  const bool many = (uint64_t)T * octets >= kManyOctets;
  const uint32_t log2 = many ? std::max(2u, ceil_log2((octets + kHeldOctets - 1) / kHeldOctets)) : std::min(8u, ceil_log2(octets));
  const uint32_t held = (octets + (1u << log2) - 1) >> log2;
  auto with = [&](auto v) {
    constexpr uint32_t V = decltype(v)::value;
    if (many)
      go(v, integral_constant<uint32_t, kHeldOctets / V>{}, log2);
    else
      go(v, integral_constant<uint32_t, 1>{}, log2);
  };
  if (held <= 1)
    with(integral_constant<uint32_t, 1>{});
  else if (held <= 2)
    with(integral_constant<uint32_t, 2>{});
  else if (held <= 4)
    with(integral_constant<uint32_t, 4>{});
  else
    with(integral_constant<uint32_t, 8>{});
}

template <class Y>
void dequantize(const void *codes, const void *scales, uint32_t R, uint32_t K, void *out, cudaStream_t st) {
  const uint32_t octets = K / 8, log2 = std::min(8u, ceil_log2(octets)), pieces = (octets + (1u << log2) - 1) >> log2;
  auto go = [&](auto u) {
    constexpr uint32_t U = decltype(u)::value;
    const uint32_t rows = U * (kThreads >> log2);
    CUDA_OK(launch_kernel(true, k_i8_dequantize<Y, U>, dim3((R + rows - 1) / rows, pieces), dim3(kThreads), 0, st, (const uint8_t *)codes, (const float *)scales,
                          RowsOfThreads{R, log2, octets}, K, (Y *)out));
  };
  if ((uint64_t)R * octets >= kManyOctets)
    go(std::integral_constant<uint32_t, 4>{});
  else
    go(std::integral_constant<uint32_t, 1>{});
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
