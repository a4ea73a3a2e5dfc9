// Products of MX rows in expert order with their experts' MX matrices (include/moe_layer.h: moe_mx4_product_device, moe_mx4_gate_up_device).
//
// A CTA of 256 threads takes 64 rows of one expert and 64 of its matrix's rows; 32 values of both a step are decoded to f32 in
// shared memory and every thread adds up 4 x 4 sums. For gate_up the 64 matrix rows are 32 gate rows and the 32 up rows of the same
// features, one block of h.
#include <cuda_runtime.h>

#include <cstdint>

#include "mx4.cuh"
#include "ops_common.h"

namespace moe {
namespace {

constexpr uint32_t kMaxExperts = 512;
constexpr uint32_t kTile = 64;

struct Mx4Args {
  const uint8_t *wc, *ws, *xc, *xs;
  const int32_t *offsets;
  uint32_t E, N, K, R;
  float limit;
  void *y;
  uint32_t bf16;
  uint8_t *hc, *hs;
};

// Tile `at` of the experts' rows cut into tiles of kTile: by one warp, every lane leaves with it; count 0 past the last.
__device__ __forceinline__ void find_tile(const Mx4Args &a, uint32_t at, uint32_t lane, uint32_t &expert, uint32_t &start, uint32_t &count) {
  count = 0, expert = 0, start = 0;
  for (uint32_t e0 = 0; e0 < a.E; e0 += 32) {
    const uint32_t e = e0 + lane;
    uint32_t lo = 0, n = 0;
    if (e < a.E) {
      lo = a.offsets ? min((uint32_t)max(a.offsets[e], 0), a.R) : 0u;
      const uint32_t hi = a.offsets ? min((uint32_t)max(a.offsets[e + 1], 0), a.R) : a.R;
      n = hi > lo ? hi - lo : 0;
    }
    const uint32_t nt = (n + kTile - 1) / kTile;
    uint32_t upto = nt;
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= (uint32_t)off) upto += o;
    }
    const uint32_t here = __ballot_sync(0xffffffffu, at < upto);
    if (here) {
      const int l = __ffs(here) - 1;
      const uint32_t skip = at - (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, nt, l));
      expert = e0 + l, start = __shfl_sync(0xffffffffu, lo, l) + skip * kTile;
      count = min(kTile, __shfl_sync(0xffffffffu, n, l) - skip * kTile);
      return;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <bool GU>
__global__ void __launch_bounds__(256) k_mx4_simple(const Mx4Args a) {
  __shared__ float xt[32][kTile + 4], wt[32][kTile + 4];
  __shared__ float o[GU ? kTile : 1][GU ? kTile + 1 : 1];
  __shared__ uint32_t s_tile[3];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t tid = threadIdx.x;
  if (tid < 32) {
    uint32_t e, s, c;
    find_tile(a, blockIdx.y, tid, e, s, c);
    if (tid == 0) s_tile[0] = e, s_tile[1] = s, s_tile[2] = c;
  }
  __syncthreads();
  const uint32_t expert = s_tile[0], start = s_tile[1], count = s_tile[2];
  if (!count) return;
  const uint32_t F = a.N / 2, srow = mx_scale_row_bytes(a.K);
  // Loads: row tid / 4 of the tile, eight values at 8 (tid % 4).
  const uint32_t lr = tid / 4, lk = tid % 4 * 8;
  const bool xin = lr < count;
  const uint64_t xr = start + lr;
  const uint32_t n0 = blockIdx.x * (GU ? 32 : kTile), wn = GU ? (lr < 32 ? n0 + lr : F + n0 + lr - 32) : n0 + lr;
  const bool win = GU || wn < a.N;
  const uint64_t wr = (uint64_t)expert * a.N + wn;
  float acc[4][4] = {};
  const uint32_t ty = tid / 16, tx = tid % 16;
  for (uint32_t k = 0; k < a.K; k += 32) {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (xin) {
      mx_values8(*(const uint32_t *)(a.xc + xr * (a.K / 2) + (k + lk) / 2), v);
      const float f = mx_scale(a.xs[xr * srow + k / 32]);
      for (int i = 0; i < 8; i++) v[i] *= f;
    }
    if (win) {
      mx_values8(*(const uint32_t *)(a.wc + wr * (a.K / 2) + (k + lk) / 2), u);
      const float f = mx_scale(a.ws[wr * srow + k / 32]);
      for (int i = 0; i < 8; i++) u[i] *= f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) xt[lk + i][lr] = v[i], wt[lk + i][lr] = u[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; i++)
#pragma unroll
      for (int p = 0; p < 4; p++)
#pragma unroll
        for (int q = 0; q < 4; q++) acc[p][q] = fmaf(xt[i][ty * 4 + p], wt[i][tx * 4 + q], acc[p][q]);
  }
  if constexpr (!GU) {
    for (int p = 0; p < 4; p++)
      for (int q = 0; q < 4; q++) {
        const uint32_t r = ty * 4 + p, n = n0 + tx * 4 + q;
        if (r >= count || n >= a.N) continue;
        const uint64_t at = (uint64_t)(start + r) * a.N + n;
        if (a.bf16)
          ((__nv_bfloat16 *)a.y)[at] = __float2bfloat16_rn(acc[p][q]);
        else
          ((__half *)a.y)[at] = __float2half_rn(acc[p][q]);
      }
  } else {
    for (int p = 0; p < 4; p++)
      for (int q = 0; q < 4; q++) o[ty * 4 + p][tx * 4 + q] = acc[p][q];
    __syncthreads();
    float h[8];
    uint32_t m = 0;
    for (int i = 0; i < 8; i++) {
      float g = o[lr][lk + i], u = o[lr][32 + lk + i];
      if (a.limit > 0.0f) g = fminf(g, a.limit), u = fminf(fmaxf(u, -a.limit), a.limit);
      h[i] = g / (1.0f + expf(-g)) * u;
      m = max(m, __float_as_uint(h[i]) & 0x7FFFFFFFu);
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t scale = mx_scale_of(m);
    const float f = mx_inverse(scale);
    for (int i = 0; i < 8; i++) h[i] *= f;
    if (lr < count) {
      const uint64_t r = start + lr;
      const uint32_t hrow = mx_scale_row_bytes(F);
      *(uint32_t *)(a.hc + r * (F / 2) + (n0 + lk) / 2) = scale == 255 ? 0u : mx_codes8(h);
      if (tid % 4 == 0) a.hs[r * hrow + n0 / 32] = (uint8_t)scale;
      if (tid % 4 == 0 && n0 + 32 == F)
        for (uint32_t b = F / 32; b < hrow; b++) a.hs[r * hrow + b] = 0;
    }
  }
}

Mx4Args arguments(const moe_mx4_weights *w, const void *codes, const void *scales, uint32_t R, const int32_t *offsets) {
  need(w != nullptr, "weights are required");
  need(w->n_experts >= 1 && w->n_experts <= kMaxExperts, "n_experts must be 1 .. 512");
  need(w->n_out >= 32 && w->n_out % 32 == 0 && w->n_out <= kMxMaxValues, "n_out must be a multiple of 32, 32 .. 65536");
  need(w->n_in >= 32 && w->n_in % 32 == 0 && w->n_in <= kMxMaxValues, "n_in must be a multiple of 32, 32 .. 65536");
  need(w->reserved == 0, "reserved must be 0");
  need(offsets || w->n_experts == 1, "offsets are required for more than one expert");
  need(R <= 1u << 24, "R must be at most 2^24");
  Mx4Args a{};
  a.wc = (const uint8_t *)w->codes_dev, a.ws = (const uint8_t *)w->scales_dev, a.xc = (const uint8_t *)codes, a.xs = (const uint8_t *)scales;
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
    Mx4Args a = arguments(w, codes_dev, scales_dev, R, offsets_dev);
    if (R == 0) return;
    need_device({{a.wc, "weight codes", 16}, {a.ws, "weight scales", 4}, {a.xc, "codes", 16}, {a.xs, "scales", 4}, {a.offsets, "offsets", 4, true}, {y_dev, "y", 16}});
    a.y = y_dev, a.bf16 = y_type == MOE_TYPE_BF16;
    CUDA_OK(launch_kernel(true, k_mx4_simple<false>, dim3((a.N + kTile - 1) / kTile, R / kTile + a.E), dim3(256), 0, (cudaStream_t)stream, a));
  });
}

MOE_API moe_status moe_mx4_gate_up_device(const moe_mx4_weights *w, const void *codes_dev, const void *scales_dev, uint32_t R,
                                          const int32_t *offsets_dev, float swiglu_limit, void *h_codes_dev, void *h_scales_dev, void *stream) {
  return ops_call([&] {
    need(!(swiglu_limit < 0.0f) && swiglu_limit - swiglu_limit == 0.0f, "swiglu_limit must be 0 or a positive number");
    Mx4Args a = arguments(w, codes_dev, scales_dev, R, offsets_dev);
    need(a.N % 64 == 0, "gate and up rows together must be a multiple of 64");
    if (R == 0) return;
    need_device({{a.wc, "weight codes", 16}, {a.ws, "weight scales", 4}, {a.xc, "codes", 16}, {a.xs, "scales", 4}, {a.offsets, "offsets", 4, true},
                 {h_codes_dev, "h codes", 16}, {h_scales_dev, "h scales", 4}});
    a.limit = swiglu_limit, a.hc = (uint8_t *)h_codes_dev, a.hs = (uint8_t *)h_scales_dev;
    CUDA_OK(launch_kernel(true, k_mx4_simple<true>, dim3(a.N / 64, R / kTile + a.E), dim3(256), 0, (cudaStream_t)stream, a));
  });
}

}  // extern "C"
