// Two f32 numbers that one instruction takes together (fma.rn.f32x2 and mul.rn.f32x2 of sm_100), each rounded as by itself.
#pragma once

#include <cstdint>

namespace moe {

struct Two {
  uint64_t v;
  Two() = default;
  __device__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ explicit Two(float a) : Two(a, a) {}
  __device__ float lo() const { return __uint_as_float((uint32_t)v); }
  __device__ float hi() const { return __uint_as_float((uint32_t)(v >> 32)); }
};
__device__ __forceinline__ Two fma(const Two &a, const Two &b, const Two &c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two operator*(const Two &a, const Two &b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator+(const Two &a, const Two &b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

}  // namespace moe
