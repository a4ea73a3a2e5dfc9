// Microscaled 4-bit floating point on the device (include/moe_layer.h, "MX rows"): e2m1 codes two a byte, an e8m0 scale every 32 values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace moe {

constexpr uint32_t kMxBlock = 32;
constexpr uint32_t kMxMaxValues = 65536;  // of a row

__host__ __device__ constexpr uint32_t mx_scale_row_bytes(uint32_t K) { return (K / kMxBlock + 3) / 4 * 4; }

#if defined(__CUDACC__)
// The scale byte of a block whose largest magnitude has these bits: floor(log2) - 2, biased by 127, from the exponent field itself.
// Below 2^-125 it stays 0 (2^-127); an infinity or NaN gives 255.
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t max_bits) {
  const uint32_t f = max_bits >> 23;
  return f == 255 ? 255u : f > 2 ? f - 2 : 0u;
}
// 2^(127 - byte): what the values are multiplied by, exactly, before they are rounded. 0 for byte 255, whose codes are 0.
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return byte == 255 ? 0.0f : __uint_as_float((254 - byte) << 23); }
// 2^(byte - 127); NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7FFFFFFFu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// Eight values to codes, the first in the lowest four bits: to nearest, ties to even, beyond 6 to 6.
__device__ __forceinline__ uint32_t mx_codes8(const float *v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// The eight codes' values.
__device__ __forceinline__ void mx_values8(uint32_t codes, float *v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*(const __half2 *)&h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
// Eight values of a row, 16-byte aligned, as f32.
__device__ __forceinline__ void load8(const float *p, float *v) {
  *(float4 *)v = *(const float4 *)p, *(float4 *)(v + 4) = *(const float4 *)(p + 4);
}
__device__ __forceinline__ void load8(const __half *p, float *v) {
  const uint4 u = *(const uint4 *)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*(const __half2 *)&w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float *v) {
  const uint4 u = *(const uint4 *)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void store8(float *p, const float *v) { *(float4 *)p = *(const float4 *)v, *(float4 *)(p + 4) = *(const float4 *)(v + 4); }
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half *) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t *)&h;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16 *) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t *)&h;
}
template <class Y>
__device__ __forceinline__ void store8(Y *p, const float *v) {
  *(uint4 *)p = make_uint4(pack2(v[0], v[1], p), pack2(v[2], v[3], p), pack2(v[4], v[5], p), pack2(v[6], v[7], p));
}
#endif

}  // namespace moe
