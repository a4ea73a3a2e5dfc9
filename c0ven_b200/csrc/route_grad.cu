// The gradient of the routing's weights (moe_route_logits_device) with respect to the logits, the chosen experts held fixed.
//
// With s an expert's score, K a row's chosen experts, c the weights' factor, d the weights' gradient and m = sum over K of p d:
//   softmax, renormalised: p = e^l / sum over K,      dl = c p (d - m) in K, 0 elsewhere;
//   softmax as it is:      p = e^l / sum over all,    dl = c p (d - m), d 0 outside K;
//   sigmoid, renormalised: p = s / sum of s over K,   dl = c p (1 - s) (d - m) in K, 0 elsewhere;
//   sigmoid as it is:                                 dl = c s (1 - s) d in K, 0 elsewhere.
//
// A warp takes a row; its lanes 0 .. n_used - 1 an assignment each, then every lane its columns of the row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ops_common.h"

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

// V: columns a lane has at most.
template <class L, int V>
__global__ void __launch_bounds__(32 * kWarps) k_route_grad(const RouteGradArgs a) {
  __shared__ float rows[kWarps][32 * V];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint64_t t = (uint64_t)blockIdx.x * kWarps + warp;
  if (t >= a.T) return;
  float *row = rows[warp];
  uint32_t id = 0xFFFFFFFFu;
  float d = 0.0f, l = -INFINITY;
  if (lane < a.k) {
    id = (uint32_t)a.ids[t * a.k + lane];
    if (id < a.E) d = a.dw[t * a.k + lane], l = logit_of<L>(a, t, id);
    if (l == -INFINITY) d = 0.0f;
  }
  const bool dense = !a.sigmoid && !a.renorm;
  float z[V];
  if (dense) {
#pragma unroll
    for (int v = 0; v < V; v++) z[v] = lane + 32 * v < a.E ? logit_of<L>(a, t, lane + 32 * v) : -INFINITY;
  }
#pragma unroll
  for (int v = 0; v < V; v++) row[lane + 32 * v] = 0.0f;
  __syncwarp();
  if (dense) {
    float top = z[0];
#pragma unroll
    for (int v = 1; v < V; v++) top = fmaxf(top, z[v]);
    top = warp_max(top);
    float total = 0.0f;
#pragma unroll
    for (int v = 0; v < V; v++) z[v] = part_of(z[v], top), total += z[v];
    total = warp_sum(total);
    const float mean = total > 0.0f ? warp_sum(part_of(l, top) * d) / total : 0.0f, f = total > 0.0f ? a.scale / total : 0.0f;
    if (id < a.E) row[id] = d;
    __syncwarp();
#pragma unroll
    for (int v = 0; v < V; v++) z[v] = f * z[v] * (row[lane + 32 * v] - mean);
  } else {
    const float top = warp_max(l);
    float p = 0.0f, rest = 1.0f;  // rest: 1 - s
    if (a.sigmoid) {
      rest = 1.0f / (1.0f + expf(l));
      // Relative to the largest where all scores are small: from e^-60 on they are e^l to f32.
      p = l == -INFINITY ? 0.0f : a.renorm && top < -60.0f ? part_of(l, top) : 1.0f / (1.0f + expf(-l));
    } else {
      p = part_of(l, top);
    }
    if (a.renorm) {
      const float total = warp_sum(p);
      p = total > 0.0f ? p / total : 0.0f;
      const float mean = warp_sum(p * d);
      if (id < a.E) row[id] = a.scale * p * rest * (d - mean);
    } else if (id < a.E) {
      row[id] = a.scale * p * rest * d;
    }
    __syncwarp();
#pragma unroll
    for (int v = 0; v < V; v++) z[v] = row[lane + 32 * v];
  }
#pragma unroll
  for (int v = 0; v < V; v++)
    if (lane + 32 * v < a.E) ((L *)a.out)[t * a.out_stride + lane + 32 * v] = (L)z[v];
}

template <class L>
void launch_grad(const RouteGradArgs &a, cudaStream_t st) {
  const dim3 grid((a.T + kWarps - 1) / kWarps), block(32 * kWarps);
  const auto kernel = a.E <= 32 ? k_route_grad<L, 1> : a.E <= 64 ? k_route_grad<L, 2> : a.E <= 128 ? k_route_grad<L, 4> : a.E <= 256 ? k_route_grad<L, 8> : k_route_grad<L, 16>;
  CUDA_OK(launch_kernel(true, kernel, grid, block, 0, st, a));
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
