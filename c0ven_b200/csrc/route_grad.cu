// The gradient of the routing's weights (moe_route_logits_device) with respect to the logits, the chosen experts held fixed.
//
// With s an expert's score, K a row's chosen experts, c the weights' factor, d the weights' gradient and m = sum over K of p d:
//   softmax, renormalised: p = e^l / sum over K,      dl = c p (d - m) in K, 0 elsewhere;
//   softmax as it is:      p = e^l / sum over all,    dl = c p (d - m), d 0 outside K;
//   sigmoid, renormalised: p = s / sum of s over K,   dl = c p (1 - s) (d - m) in K, 0 elsewhere;
//   sigmoid as it is:                                 dl = c s (1 - s) d in K, 0 elsewhere.
//
// A warp takes a row; its lanes 0 .. n_used - 1 an assignment each, then every lane its columns of the row, which the assignments' numbers reach through shared
// memory. Softmax weights as they are read and write every logit: 32,768 rows of 512 f32 values 25 us (5.4 TB/s), of bf16 23 (2.9), bound by the
// exponentials' and reductions' instructions; 57 with an accurate exponential and a column at a time. The others read the chosen logits alone: 18.6 us for as many f32
// rows (3.7 TB/s), one dependent load after another.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ops_common.h"
#include "two.cuh"

namespace moe {
namespace {

constexpr uint32_t kMaxExperts = 512, kMaxUsed = 16, kWarps = 8;

struct RouteGradArgs {
  const void *logits;
  uint64_t stride;
  const float *bias;
  uint32_t T, E, k;
  bool sigmoid, renorm;
  float scale;
  const int32_t *ids;
  const float *dw;
  void *out;
  uint64_t out_stride;
};

// The expert's logit, -infinity if it is out.
template <class L>
__device__ __forceinline__ float logit_of(const RouteGradArgs &a, uint64_t t, uint32_t e) {
  const float l = (float)((const L *)a.logits)[t * a.stride + e];
  return l > -INFINITY && (!a.bias || a.bias[e] > -INFINITY) ? l : -INFINITY;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off; off /= 2) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off; off /= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
// e^(l - top), the largest's own 1 even where it is infinite; 0 for an expert that is out.
__device__ __forceinline__ float part_of(float l, float top) { return l == -INFINITY ? 0.0f : l == top ? 1.0f : expf(l - top); }
constexpr float kLog2e = 1.4426950408889634f;
// A row's largest logit from which on its product with log2(e) might be rounded by what 2^ of passes f32: by 1/16 below.
constexpr float kFarTop = 0x1p20f;
// f d, 0 for a factor that vanished whatever d is: a weight's gradient that is no number reaches no expert by a share of 0.
__device__ __forceinline__ float weighed(float f, float d) { return f != 0.0f ? f * d : 0.0f; }
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Four neighbouring values of a row as f32, and back. The address is aligned to them.
__device__ __forceinline__ void load4(const float *p, float *v) { *(float4 *)v = *(const float4 *)p; }
__device__ __forceinline__ void load4(const __half *p, float *v) {
  const uint2 u = *(const uint2 *)p;
  *(float2 *)v = __half22float2(*(const __half2 *)&u.x), *(float2 *)(v + 2) = __half22float2(*(const __half2 *)&u.y);
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *v) {
  const uint2 u = *(const uint2 *)p;
  v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xFFFF0000u), v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
__device__ __forceinline__ void store4(float *p, const float *v) { *(float4 *)p = *(const float4 *)v; }
__device__ __forceinline__ void store4(__half *p, const float *v) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *(uint2 *)p = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float *v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *(uint2 *)p = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
}

// CTAs an SM. Softmax weights as they are: as many as are resident at once, whose warps bring their next row while they work on one, with registers for three (32,768
// rows of 512 f32 logits: 25 us, 30 without that bound and with six CTAs an SM, 34 with two resident and three launched; the bytes alone 20.5). Else a row
// is short work (32,768 rows of 512 f32 values 19 us, of 256 bf16 ones 12.6 with 16 an SM, 19 and 12.7 with 8, 19 and 13.4 with 28).
template <int V, bool DENSE>
constexpr uint32_t grad_ctas() {
  return !DENSE ? 16 : V == 16 ? 3 : V == 8 ? 4 : 6;
}

// V: columns a lane has at most. W: neighbouring ones it has together, four where the rows' addresses allow, else one. DENSE: softmax weights as they are.
template <class L, int V, int W, bool DENSE>
__global__ void __launch_bounds__(32 * kWarps, DENSE ? grad_ctas<V, DENSE>() : 8) k_route_grad(const RouteGradArgs a) {
  __shared__ __align__(16) float rows[kWarps][32 * V];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  float *row = rows[warp];
  auto column = [&](int v) { return v / W * 32 * W + lane * W + v % W; };
#pragma unroll
  for (int v = 0; v < V; v++) row[column(v)] = 0.0f;
  __syncwarp();
  // An assignment a lane, and for softmax weights as they are the row's logits: of the warp's next row while this one is worked on.
  uint32_t id = 0xFFFFFFFFu;
  float d = 0.0f, l = -INFINITY, z[DENSE ? V : 1];
  auto bring = [&](uint64_t t) {
    id = 0xFFFFFFFFu, d = 0.0f, l = -INFINITY;
    if (lane < a.k) {
      id = (uint32_t)a.ids[t * a.k + lane];
      if (id < a.E) d = a.dw[t * a.k + lane];
      if (!DENSE && id < a.E) l = logit_of<L>(a, t, id);
    }
    if constexpr (DENSE) {
      const L *p = (const L *)a.logits + t * a.stride;
#pragma unroll
      for (int v = 0; v < V; v += W) {
        if constexpr (W == 4) {
          if (column(v) < a.E)
            load4(p + column(v), z + v);
          else
            z[v] = z[v + 1] = z[v + 2] = z[v + 3] = -INFINITY;
        } else {
          z[v] = column(v) < a.E ? (float)p[column(v)] : -INFINITY;
        }
      }
    }
  };
  const uint64_t step = (uint64_t)gridDim.x * kWarps;
  uint64_t t = (uint64_t)blockIdx.x * kWarps + warp;
  if (t < a.T) bring(t);
  for (; t < a.T; t += step) {
    const uint32_t e = id;
    float y[V], g = d;
    if constexpr (DENSE) {
      // An expert that is out, NaN among them, counts as -infinity. The exponentials are 2^(l log2(e) - top log2(e)), approximate, off by 2^-22 and by the argument's one
      // rounding and its factor's, 1.22 parts in 2^24 of l - top: some more than rounding l - top does to an accurate one. How the second product was rounded is
      // one factor of the whole row, which its shares do not have.
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < V; v++) {
        y[v] = fmaxf(z[v], -INFINITY);
        if (a.bias && column(v) < a.E && !(a.bias[column(v)] > -INFINITY)) y[v] = -INFINITY;
        top = fmaxf(top, y[v]);
      }
      if (e < a.E) row[e] = g;
      const bool odd = __any_sync(0xffffffffu, !(fabsf(g) < 1e30f));
      if (t + step < a.T) bring(t + step);
      top = warp_max(top);
      if (!(fabsf(top) < kFarTop)) {
#pragma unroll
        for (int v = 0; v < V; v++) y[v] = top == INFINITY ? (y[v] == INFINITY ? 0.0f : -INFINITY) : top == -INFINITY ? y[v] : y[v] - top;  // infinite ones alone share the row
        top = 0.0f;
      }
      const Two log2e(kLog2e), less(-top * kLog2e);
      Two total(0.0f);
#pragma unroll
      for (int v = 0; v < V; v += 2) {
        const Two p = fma(Two(y[v], y[v + 1]), log2e, less);
        y[v] = exp2_approx(p.lo()), y[v + 1] = exp2_approx(p.hi());
        total = total + Two(y[v], y[v + 1]);
      }
      const float sum = warp_sum(total.lo() + total.hi());
      __syncwarp();
      Two part(0.0f);
      float c[V];
#pragma unroll
      for (int v = 0; v < V; v++) c[v] = row[column(v)];
      if (odd) {  // a weight's gradient that is no number reaches those that its expert's share does; one so large is weighed before it is summed
        float m = 0.0f;
#pragma unroll
        for (int v = 0; v < V; v++) m += y[v] > 0.0f ? y[v] / sum * c[v] : 0.0f;
        const float mean = warp_sum(m);
#pragma unroll
        for (int v = 0; v < V; v++) y[v] = y[v] > 0.0f ? weighed(a.scale / sum * y[v], c[v] - mean) : 0.0f;
      } else {
#pragma unroll
        for (int v = 0; v < V; v += 2) part = fma(Two(y[v], y[v + 1]), Two(c[v], c[v + 1]), part);
        const float f = sum > 0.0f ? a.scale / sum : 0.0f, mean = sum > 0.0f ? warp_sum(part.lo() + part.hi()) / sum : 0.0f;
        const Two factor(f), minus(-mean);
#pragma unroll
        for (int v = 0; v < V; v += 2) {
          const Two r = (Two(c[v], c[v + 1]) + minus) * (Two(y[v], y[v + 1]) * factor);
          y[v] = r.lo(), y[v + 1] = r.hi();
        }
      }
    } else {
      const float lc = l;
      if (lc == -INFINITY) g = 0.0f;
      if (t + step < a.T) bring(t + step);
      const float top = warp_max(lc);
      float p = 0.0f, rest = 1.0f;  // rest: 1 - s
      if (a.sigmoid) {
        rest = 1.0f / (1.0f + expf(lc));
        // Relative to the largest where all scores are small: from e^-60 on they are e^l to f32.
        p = lc == -INFINITY ? 0.0f : a.renorm && top < -60.0f ? part_of(lc, top) : 1.0f / (1.0f + expf(-lc));
      } else {
        p = part_of(lc, top);
      }
      if (a.renorm) {
        const float total = warp_sum(p);
        p = total > 0.0f ? p / total : 0.0f;
        g -= warp_sum(weighed(p, g));
      }
      if (e < a.E) row[e] = weighed(a.scale * p * rest, g);
      __syncwarp();
#pragma unroll
      for (int v = 0; v < V; v++) y[v] = row[column(v)];
    }
    L *out = (L *)a.out + t * a.out_stride;
#pragma unroll
    for (int v = 0; v < V; v += W) {
      if constexpr (W == 4) {
        if (column(v) < a.E) store4(out + column(v), y + v);
      } else {
        if (column(v) < a.E) out[column(v)] = (L)y[v];
      }
    }
    __syncwarp();
    if (e < a.E) row[e] = 0.0f;
    __syncwarp();
  }
}

template <class L, int V, int W, bool DENSE>
void launch_columns(const RouteGradArgs &a, cudaStream_t st) {
  const dim3 grid(std::min((a.T + kWarps - 1) / kWarps, 148 * grad_ctas<V, DENSE>())), block(32 * kWarps);
  CUDA_OK(launch_kernel(true, k_route_grad<L, V, W, DENSE>, grid, block, 0, st, a));
}

template <class L, int W, bool DENSE>
void launch_grad(const RouteGradArgs &a, cudaStream_t st) {
  if (a.E <= 128)
    launch_columns<L, 4, W, DENSE>(a, st);
  else if (a.E <= 256)
    launch_columns<L, 8, W, DENSE>(a, st);
  else
    launch_columns<L, 16, W, DENSE>(a, st);
}

template <class L>
void launch_grad(const RouteGradArgs &a, cudaStream_t st) {
  const uint64_t at = (uint64_t)a.logits | (uint64_t)a.out | a.stride * sizeof(L) | a.out_stride * sizeof(L);
  const bool dense = !a.sigmoid && !a.renorm, four = a.E % 4 == 0 && at % (4 * sizeof(L)) == 0;
  const auto call = dense ? (four ? launch_grad<L, 4, true> : launch_grad<L, 1, true>) : (four ? launch_grad<L, 4, false> : launch_grad<L, 1, false>);
  call(a, st);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API moe_status moe_route_logits_grad_device(const moe_route_config *config, const void *logits_dev, uint64_t stride, const float *bias_dev, uint32_t T,
                                                const int32_t *ids_dev, const float *dw_dev, void *dlogits_dev, uint64_t dlogits_stride, void *stream) {
  return ops_call([&] {
    need(config != nullptr, "config is required");
    const moe_route_config &c = *config;
    need(c.n_experts >= 1 && c.n_experts <= kMaxExperts, "n_experts must be 1 .. 512");
    need(c.n_used >= 1 && c.n_used <= kMaxUsed && c.n_used <= c.n_experts, "n_used must be 1 .. 16 and at most n_experts");
    need(c.score <= MOE_SCORE_SIGMOID, "score must be MOE_SCORE_SOFTMAX or MOE_SCORE_SIGMOID");
    const uint32_t size = row_type_bytes(c.logits_type);
    need(size != 0, "logits_type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need(c.scale - c.scale == 0.0f, "scale must be finite");
    need(stride == 0 || (stride >= c.n_experts && stride < 1ull << 32), "stride must be 0, or n_experts at least");
    need(dlogits_stride == 0 || (dlogits_stride >= c.n_experts && dlogits_stride < 1ull << 32), "dlogits_stride must be 0, or n_experts at least");
    need(T <= 1u << 24, "T must be at most 2^24");
    if (T == 0) return;
    need_device({{logits_dev, "logits", size}, {bias_dev, "bias", 4, true}, {ids_dev, "ids", 4}, {dw_dev, "dw", 4}, {dlogits_dev, "dlogits", size}});
    const RouteGradArgs a{logits_dev, stride ? stride : c.n_experts, bias_dev, T, c.n_experts, c.n_used, c.score == MOE_SCORE_SIGMOID, c.no_renorm == 0,
                          c.scale == 0.0f ? 1.0f : c.scale, ids_dev, dw_dev, dlogits_dev, dlogits_stride ? dlogits_stride : c.n_experts};
    if (c.logits_type == MOE_TYPE_F32)
      launch_grad<float>(a, (cudaStream_t)stream);
    else if (c.logits_type == MOE_TYPE_F16)
      launch_grad<__half>(a, (cudaStream_t)stream);
    else
      launch_grad<__nv_bfloat16>(a, (cudaStream_t)stream);
  });
}

}  // extern "C"
