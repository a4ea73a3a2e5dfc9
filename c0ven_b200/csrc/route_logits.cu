// Routing of a step's logits without a layer: softmax or sigmoid scores, a bias that chooses but does not weigh, groups of
// experts, the top n_used, and the lists of expert order (moe_route_logits_device).
//
// A warp takes a row; lane l holds experts l, l + 32, .... Keys (score + bias) are first worked out in f32, with the fast exponential and
// division, and the largest are taken off one at a time by a warp-wide maximum of order-preserving integers. That decides the row
// when every two neighbours among the keys taken, and the last taken and the first left, are further apart than the f32 keys'
// error (key_error): the order is then that of the exact keys. Else (two keys in some ten thousand rows of distinct logits) the warp
// takes the row again with keys in f64. Without bias and groups the scores' order is the logits' own, which are exact. The weights come from
// the chosen logits alone, by the accurate exponential, relative to the largest of them, so that they neither overflow nor
// vanish together.
//
// What bounds it: 32,768 rows of 512 f32 logits are 67 MB, 10 us of HBM; the selection's instructions take longer.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ops_common.h"

namespace moe {

std::string &ops_error() {
  thread_local std::string text;
  return text;
}

namespace {

constexpr uint32_t kRouteMaxExperts = 512, kRouteMaxUsed = 16, kRouteMaxGroups = 32;
constexpr uint32_t kRouteChunk = 32;     // rows whose experts are counted together
constexpr uint32_t kRouteWarps = 8;      // of a CTA that takes a chunk
constexpr uint32_t kRouteOneCta = 64;    // rows that one CTA of 32 warps routes and lists by itself
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct RouteArgs {
  const void *logits;
  uint64_t stride;
  const float *bias;
  uint32_t T, E, k, G, used, gsize;
  bool sigmoid, renorm;
  float scale;
  int32_t *ids;
  float *w;
  int32_t *offsets, *inv;
  uint32_t *work;  // [chunks][E] counts, then [E] totals
};

// The expert's logit, -infinity if it is out.
template <class L>
__device__ __forceinline__ float logit_of(const RouteArgs &a, uint64_t t, uint32_t e) {
  const float l = (float)((const L *)a.logits)[t * a.stride + e] + 0.0f;  // -0 is 0
  return l > -INFINITY && (!a.bias || a.bias[e] > -INFINITY) ? l : -INFINITY;
}

// f32 as an integer of the same order.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }

// Arithmetic of the keys by type. f32: the fast forms, whose errors key_error bounds. f64: what decides.
__device__ __forceinline__ float key_exp(float x) { return __expf(x); }
__device__ __forceinline__ double key_exp(double x) { return exp(x); }
__device__ __forceinline__ float key_div(float a, float b) { return __fdividef(a, b); }
__device__ __forceinline__ double key_div(double a, double b) { return a / b; }
template <class T>
__device__ __forceinline__ T minus_inf() {
  return (T)(-INFINITY);
}
template <class T>
__device__ __forceinline__ T sigmoid_key(T l) {
  const T e = key_exp(l < 0 ? l : -l);  // at most 1
  return key_div(l < 0 ? e : (T)1, (T)1 + e);
}
// e^(l - largest), the largest's own 1 even where it is infinite.
template <class T>
__device__ __forceinline__ T softmax_part(float l, float largest) {
  return l == largest ? (T)1 : key_exp((T)l - (T)largest);
}

// e^(l - c) for l <= c by the accurate exponential, what the difference's rounding left out with it (of differences near 80 that alone is
// 4e-6 of the result).
__device__ __forceinline__ float exp_below(float l, float c) {
  if (l == c) return 1.0f;
  const float d = l - c, b = d - l, lost = (l - (d - b)) + (-c - b), e = expf(d);
  return e > 0.0f ? fmaf(e, lost, e) : 0.0f;
}

// The warp's largest of (v, e), ties to the lower e; every lane leaves with it. Lanes with nothing bring -infinity and kNone.
__device__ __forceinline__ void warp_best(float &v, uint32_t &e) {
  const uint32_t m = __reduce_max_sync(0xffffffffu, ordered(v));
  e = __reduce_min_sync(0xffffffffu, ordered(v) == m ? e : kNone);
  v = unordered(m);
}
__device__ __forceinline__ void warp_best(double &v, uint32_t &e) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double ov = __shfl_xor_sync(0xffffffffu, v, off);
    const uint32_t oe = __shfl_xor_sync(0xffffffffu, e, off);
    if (ov > v || (ov == v && oe < e)) v = ov, e = oe;
  }
}

// What the f32 score of any of a row's experts may be off by. CUDA's documented bounds: the fast exponential of x is within 2 + 1.173 |x| ulp,
// the fast division within 2. A sigmoid is made of e^-|l| <= 1 with |l| e^-|l| < 0.37: 2^-20 covers it. A softmax score e^-d / sum is
// within (4 + d) 2^-22 of itself, the rounding of l - largest with it, so within 2^-20 of the largest score; and its sum, the mean of (4 + d) over
// 512 experts by their e^-d being 8 at most, within 2^-19: 2^-18 of the largest score covers both.
__device__ __forceinline__ float key_error(bool sigmoid, float largest_score) { return sigmoid ? 9.5367432e-7f : 3.8146973e-6f * largest_score; }

// Groups, on the warp's E keys in shared memory: each ranked by the sum of its two best; the keys of all but the best a.used become
// -infinity. Returns whether the choice is sure: always for f64; for f32 when the sums of the last group that stays and the first
// that goes are further apart than off, what two of them may be off by.
template <class T>
__device__ __forceinline__ bool keep_groups(T *sk, const RouteArgs &a, uint32_t lane, bool check, float off) {
  const T none = minus_inf<T>();
  // 32 / P lanes a group, P the groups rounded up to a power of two.
  uint32_t per = 32;
  while (per * a.G > 32) per >>= 1;
  const uint32_t g = lane / per;
  T one = none, two = none;
  if (g < a.G)
    for (uint32_t i = lane % per; i < a.gsize; i += per) {
      const T v = sk[g * a.gsize + i];
      if (v > one)
        two = one, one = v;
      else if (v > two)
        two = v;
    }
  for (uint32_t d = per / 2; d > 0; d >>= 1) {
    const T o1 = __shfl_xor_sync(0xffffffffu, one, d), o2 = __shfl_xor_sync(0xffffffffu, two, d);
    if (o1 > one)
      two = one > o2 ? one : o2, one = o1;
    else if (o1 > two)
      two = o1;
  }
  // A group with one expert left counts by it alone; one with none is never better than another.
  T mine = two == none ? one : one + two, last = 0;
  if (lane % per || g >= a.G) mine = none;
  uint32_t stay = 0;  // bit g: the group stays
  bool sure = true;
  for (uint32_t j = 0; j < a.used + (check ? 1 : 0); j++) {
    T v = mine;
    uint32_t best = mine > none ? g : kNone;
    warp_best(v, best);
    if (best == kNone) break;
    if (j == a.used) {
      sure = (float)(last - v) > off;
      break;
    }
    last = v;
    stay |= 1u << best;
    if (best == g) mine = none;
  }
  __syncwarp();
  if (g < a.G && !(stay >> g & 1))
    for (uint32_t i = lane % per; i < a.gsize; i += per) sk[g * a.gsize + i] = none;
  __syncwarp();
  return sure;
}

// The row in f64, where f32 leaves it open: keys in shared memory, few registers, as it is rare. Lane j < k returns the j-th expert.
template <class L>
__device__ __noinline__ uint32_t choose_f64(const RouteArgs &a, uint64_t t, uint32_t lane, float largest, double *sk) {
  double sum = 0;
  for (uint32_t e = lane; e < a.E; e += 32) {
    const float l = logit_of<L>(a, t, e);
    sk[e] = l == -INFINITY ? -INFINITY : a.sigmoid ? sigmoid_key<double>(l) : softmax_part<double>(l, largest);
    if (l > -INFINITY) sum += sk[e];
  }
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  for (uint32_t e = lane; e < a.E; e += 32) {
    if (!a.sigmoid) sk[e] /= sum;  // -infinity stays
    if (a.bias && sk[e] > -INFINITY) sk[e] += a.bias[e];
  }
  __syncwarp();
  if (a.G > 1) {
    keep_groups<double>(sk, a, lane, false, 0.0f);
    if (!a.bias)  // within the groups that stay the order is the logits' own
      for (uint32_t e = lane; e < a.E; e += 32)
        if (sk[e] > -INFINITY) sk[e] = logit_of<L>(a, t, e);
    __syncwarp();
  }
  uint32_t id = kNone;
  for (uint32_t j = 0; j < a.k; j++) {
    double v = -INFINITY;
    uint32_t best = kNone;
    for (uint32_t e = lane; e < a.E; e += 32)
      if (sk[e] > v) v = sk[e], best = e;
    warp_best(v, best);
    if (best == kNone) break;
    if (lane == j) id = best;
    if (best % 32 == lane) sk[best] = -INFINITY;
  }
  __syncwarp();
  return id;
}

// One row, by a warp, with E doubles of shared memory of its own. Lane j < k returns the j-th expert (kNone: none) after writing ids and w.
template <class L, int V>
__device__ __forceinline__ uint32_t route_row(const RouteArgs &a, uint64_t t, uint32_t lane, double *sk) {
  float key[V], largest = -INFINITY;  // the logits, then the keys
#pragma unroll
  for (int i = 0; i < V; i++) key[i] = lane + 32 * i < a.E ? logit_of<L>(a, t, lane + 32 * i) : -INFINITY;
#pragma unroll
  for (int i = 0; i < V; i++) largest = fmaxf(largest, key[i]);
  largest = unordered(__reduce_max_sync(0xffffffffu, ordered(largest)));
  uint32_t id = kNone;
  float score_max = 1.0f;
  if (largest > -INFINITY) {
    const bool scored = a.bias || a.G > 1;
    if (!a.sigmoid && (scored || !a.renorm)) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) sum += key[i] == -INFINITY ? 0.0f : softmax_part<float>(key[i], largest);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      score_max = 1.0f / sum;
    }
    const float err = key_error(a.sigmoid, score_max);
    bool sure = true;
    if (scored) {
      float *fk = (float *)sk, top = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) {
        const uint32_t e = lane + 32 * i;
        if (key[i] == -INFINITY) {
          if (a.G > 1 && e < a.E) fk[e] = -INFINITY;
          continue;
        }
        float v = a.sigmoid ? sigmoid_key(key[i]) : softmax_part<float>(key[i], largest) * score_max;
        if (a.bias) key[i] = v += a.bias[e];
        if (a.G > 1) fk[e] = v, top = fmaxf(top, fabsf(v));
      }
      if (a.G > 1) {
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        __syncwarp();
        // Two sums of two keys, each with its own rounding, and theirs.
        sure = keep_groups<float>(fk, a, lane, true, 4 * err + 4.7683716e-7f * top);
#pragma unroll
        for (int i = 0; i < V; i++)
          if (lane + 32 * i < a.E && fk[lane + 32 * i] == -INFINITY) key[i] = -INFINITY;
        __syncwarp();
      }
    }
    // The largest keys, one at a time. With a bias no two neighbours among them, the first one left out with them, may lie within
    // what their scores and their sums' roundings may be off by (rounding keeps an order, so neighbours are all that has to be looked at).
    // Without one the keys are the logits, as they are.
    const uint32_t rounds = a.k + (a.bias ? 1 : 0);
    float last = 0.0f;
    for (uint32_t j = 0; j < rounds && sure; j++) {
      float v = -INFINITY;
      uint32_t e = kNone;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (key[i] > v) v = key[i], e = lane + 32 * i;
      warp_best(v, e);
      if (e == kNone) break;  // no expert is left
      if (a.bias && j > 0) sure = last - v > 2 * err + 2.3841858e-7f * fmaxf(fabsf(last), fabsf(v));
      last = v;
      if (lane == j && j < a.k) id = e;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (e == lane + 32 * i) key[i] = -INFINITY;
    }
    if (!sure) id = choose_f64<L>(a, t, lane, largest, sk);
  }
  // The weights: e^(l - c) and its like for the chosen, c the largest of them, so that a row's never all vanish.
  float s = 0.0f;
  const float lj = id != kNone ? logit_of<L>(a, t, id) : -INFINITY;
  if (a.renorm) {
    const float c = unordered(__reduce_max_sync(0xffffffffu, ordered(lj)));
    if (id != kNone) {
      if (!a.sigmoid)
        s = exp_below(lj, c);
      else if (c > 0.0f)
        s = lj > 0.0f ? 1.0f / (1.0f + expf(-lj)) : expf(lj) / (1.0f + expf(lj));
      else
        s = exp_below(lj, c) / (1.0f + expf(lj));
    }
    float sum = s;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (id != kNone) s = s / sum;  // the largest's own e^0 is in the sum
  } else if (id != kNone) {
    const float ex = a.sigmoid ? expf(-fabsf(lj)) : exp_below(lj, largest);
    s = !a.sigmoid ? ex * score_max : lj < 0.0f ? ex / (1.0f + ex) : 1.0f / (1.0f + ex);
  }
  if (lane < a.k) {
    a.ids[t * a.k + lane] = (int32_t)id;
    a.w[t * a.k + lane] = s * a.scale;
  }
  return id;
}

// A chunk of rows by a CTA of kRouteWarps warps; with lists, how many of its assignments each expert got.
template <class L, int V>
__global__ void __launch_bounds__(32 * kRouteWarps) k_route_rows(const RouteArgs a) {
  __shared__ double sk[kRouteWarps][32 * V];
  __shared__ uint32_t hist[kRouteMaxExperts];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (a.work) {
    for (uint32_t i = threadIdx.x; i < a.E; i += blockDim.x) hist[i] = 0;
    __syncthreads();
  }
  const uint32_t t0 = blockIdx.x * kRouteChunk, t1 = min(a.T, t0 + kRouteChunk);
  for (uint32_t t = t0 + warp; t < t1; t += kRouteWarps) {
    const uint32_t id = route_row<L, V>(a, t, lane, sk[warp]);
    if (a.work && id != kNone) atomicAdd(&hist[id], 1u);
  }
  if (a.work) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.E; i += blockDim.x) a.work[(uint64_t)blockIdx.x * a.E + i] = hist[i];
  }
}

// The chunks' counts become each expert's rows before the chunk; the totals come after the last chunk's. A CTA takes 32 experts, a
// warp a 32nd of the chunks.
__global__ void __launch_bounds__(1024) k_route_scan(uint32_t *work, uint32_t chunks, uint32_t E) {
  __shared__ uint32_t part[32][33];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, e = blockIdx.x * 32 + lane;
  const uint32_t per = (chunks + 31) / 32, c0 = min(chunks, warp * per), c1 = min(chunks, c0 + per);
  uint32_t run = 0;
  if (e < E)
    for (uint32_t c = c0; c < c1; c++) run += work[(uint64_t)c * E + e];
  part[warp][lane] = run;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t i = 0; i < warp; i++) before += part[i][lane];
  if (e >= E) return;
  run = before;
  for (uint32_t c = c0; c < c1; c++) {
    const uint32_t n = work[(uint64_t)c * E + e];
    work[(uint64_t)c * E + e] = run;
    run += n;
  }
  if (warp == 31) work[(uint64_t)chunks * E + e] = run;
}

// Exclusive sums of E <= 512 counts (thread e's in n) over a block of 512 threads or more; s: 16 words.
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t n, uint32_t *s) {
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t v = n;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= (uint32_t)off) v += o;
  }
  if (lane == 31 && warp < 16) s[warp] = v;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t i = 0; i < min(warp, 16u); i++) before += s[i];
  return before + v - n;
}

// Each assignment's row: its expert's first, the expert's rows of earlier chunks, and those before it in its own chunk. A thread an
// assignment (512 at most); CTA 0 leaves the offsets.
__global__ void __launch_bounds__(512) k_route_fill(const RouteArgs a, uint32_t chunks) {
  __shared__ uint32_t s_scan[16];
  __shared__ uint32_t s_first[kRouteMaxExperts];
  __shared__ uint16_t s_cnt[16][kRouteMaxExperts];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t i = threadIdx.x, warp = i / 32, lane = i % 32;
  const uint32_t n = i < a.E ? a.work[(uint64_t)chunks * a.E + i] : 0;
  const uint32_t first = exclusive_sum(n, s_scan);
  if (blockIdx.x == 0) {
    if (i < a.E) a.offsets[i] = (int32_t)first;
    if (i == a.E - 1) a.offsets[a.E] = (int32_t)(first + n);
  }
  for (uint32_t j = i; j < 16 * kRouteMaxExperts / 2; j += 512) ((uint32_t *)s_cnt)[j] = 0;
  if (i < a.E) s_first[i] = first + a.work[(uint64_t)blockIdx.x * a.E + i];
  const uint64_t a0 = (uint64_t)blockIdx.x * kRouteChunk * a.k;
  const uint32_t m = (min(a.T, (blockIdx.x + 1) * kRouteChunk) - blockIdx.x * kRouteChunk) * a.k;
  const uint32_t e = i < m ? (uint32_t)a.ids[a0 + i] : kNone;
  const bool valid = e < a.E;
  const uint32_t same = __match_any_sync(0xffffffffu, valid ? e : kRouteMaxExperts + lane), before = __popc(same & ((1u << lane) - 1));
  __syncthreads();
  if (valid && before == 0) s_cnt[warp][e] = (uint16_t)__popc(same);
  __syncthreads();
  if (i < a.E) {
    uint32_t run = 0;
    for (uint32_t w = 0; w < 16; w++) {
      const uint32_t c = s_cnt[w][i];
      s_cnt[w][i] = (uint16_t)run;
      run += c;
    }
  }
  __syncthreads();
  if (i < m) a.inv[a0 + i] = valid ? (int32_t)(s_first[e] + s_cnt[warp][e] + before) : -1;
}

// A short step by one CTA of 32 warps: rows, counts, offsets and places in one launch. Dynamic shared memory: 32 V doubles a warp, or
// the warps' counts.
template <class L, int V>
__global__ void __launch_bounds__(1024) k_route_short(const RouteArgs a) {
  extern __shared__ double s_dyn[];
  __shared__ uint32_t s_ids[kRouteOneCta * kRouteMaxUsed], s_scan[16], s_first[kRouteMaxExperts];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t i = threadIdx.x, warp = i / 32, lane = i % 32;
  for (uint32_t t = warp; t < a.T; t += 32) {
    const uint32_t id = route_row<L, V>(a, t, lane, s_dyn + warp * 32 * V);
    if (lane < a.k) s_ids[t * a.k + lane] = id;
  }
  if (!a.offsets) return;
  __syncthreads();
  uint16_t *s_cnt = (uint16_t *)s_dyn;  // [32][E]
  for (uint32_t j = i; j < 32 * a.E; j += 1024) s_cnt[j] = 0;
  const uint32_t m = a.T * a.k, e = i < m ? s_ids[i] : kNone;
  const bool valid = e < a.E;
  const uint32_t same = __match_any_sync(0xffffffffu, valid ? e : kRouteMaxExperts + lane), before = __popc(same & ((1u << lane) - 1));
  __syncthreads();
  if (valid && before == 0) s_cnt[warp * a.E + e] = (uint16_t)__popc(same);
  __syncthreads();
  uint32_t run = 0;
  if (i < a.E)
    for (uint32_t w = 0; w < 32; w++) {
      const uint32_t c = s_cnt[w * a.E + i];
      s_cnt[w * a.E + i] = (uint16_t)run;
      run += c;
    }
  const uint32_t first = exclusive_sum(run, s_scan);
  if (i < a.E) a.offsets[i] = (int32_t)first, s_first[i] = first;
  if (i == a.E - 1) a.offsets[a.E] = (int32_t)(first + run);
  __syncthreads();
  if (i < m) a.inv[i] = valid ? (int32_t)(s_first[e] + s_cnt[warp * a.E + e] + before) : -1;
}

__global__ void __launch_bounds__(512) k_route_empty(int32_t *offsets, uint32_t n) {
  dependents_may_launch(), wait_for_predecessors();
  for (uint32_t i = threadIdx.x; i < n; i += 512) offsets[i] = 0;
}

template <class L, int V>
void launch_rows(const RouteArgs &a, int device, cudaStream_t st) {
  if (a.T <= kRouteOneCta) {
    constexpr size_t smem = 32 * 32 * V * sizeof(double);  // 32 warps' keys; the counts, 64 V bytes a warp, lie in it too
    static std::atomic<uint32_t> done{0};
    CUDA_OK(ensure_dynamic_smem(k_route_short<L, V>, smem, done, device));
    CUDA_OK(launch_kernel(true, k_route_short<L, V>, dim3(1), dim3(1024), smem, st, a));
    return;
  }
  const uint32_t chunks = (a.T + kRouteChunk - 1) / kRouteChunk;
  CUDA_OK(launch_kernel(true, k_route_rows<L, V>, dim3(chunks), dim3(32 * kRouteWarps), 0, st, a));
  if (!a.offsets) return;
  CUDA_OK(launch_kernel(true, k_route_scan, dim3((a.E + 31) / 32), dim3(1024), 0, st, a.work, chunks, a.E));
  CUDA_OK(launch_kernel(true, k_route_fill, dim3(chunks), dim3(512), 0, st, a, chunks));
}

template <class L>
void launch_route(const RouteArgs &a, int device, cudaStream_t st) {
  if (a.E <= 32)
    launch_rows<L, 1>(a, device, st);
  else if (a.E <= 64)
    launch_rows<L, 2>(a, device, st);
  else if (a.E <= 128)
    launch_rows<L, 4>(a, device, st);
  else if (a.E <= 256)
    launch_rows<L, 8>(a, device, st);
  else
    launch_rows<L, 16>(a, device, st);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API const char *moe_ops_error(void) { return ops_error().c_str(); }

MOE_API uint64_t moe_route_work_bytes(uint32_t T, uint32_t n_experts) { return 4ull * n_experts * (((uint64_t)T + kRouteChunk - 1) / kRouteChunk + 1); }

MOE_API moe_status moe_route_logits_device(const moe_route_config *config, const void *logits_dev, uint64_t stride, const float *bias_dev,
                                           uint32_t T, int32_t *ids_dev, float *w_dev, int32_t *offsets_dev, int32_t *inv_dev,
                                           void *work_dev, uint64_t work_bytes, void *stream) {
  return ops_call([&] {
    need(config != nullptr, "config is required");
    const moe_route_config &c = *config;
    need(c.n_experts >= 1 && c.n_experts <= kRouteMaxExperts, "n_experts must be 1 .. 512");
    need(c.n_used >= 1 && c.n_used <= kRouteMaxUsed && c.n_used <= c.n_experts, "n_used must be 1 .. 16 and at most n_experts");
    need(c.score <= MOE_SCORE_SIGMOID, "score must be MOE_SCORE_SOFTMAX or MOE_SCORE_SIGMOID");
    const uint32_t G = std::max(1u, c.n_groups), size = row_type_bytes(c.logits_type);
    need(G <= kRouteMaxGroups && c.n_experts % G == 0, "n_groups must divide n_experts and be at most 32");
    if (G > 1)
      need(c.n_groups_used >= 1 && c.n_groups_used <= G && c.n_groups_used * (c.n_experts / G) >= c.n_used,
           "n_groups_used must be 1 .. n_groups, and those groups hold n_used experts");
    need(size != 0, "logits_type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need(c.scale - c.scale == 0.0f, "scale must be finite");
    need(stride == 0 || (stride >= c.n_experts && stride < 1ull << 32), "stride must be 0, or n_experts at least");
    need(T <= 1u << 24, "T must be at most 2^24");
    need((offsets_dev == nullptr) == (inv_dev == nullptr), "offsets and inv come together");
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
      need_device({{offsets_dev, "offsets", 4, true}});
      if (offsets_dev) CUDA_OK(launch_kernel(true, k_route_empty, dim3(1), dim3(512), 0, st, offsets_dev, c.n_experts + 1));
      return;
    }
    const bool lists = offsets_dev && T > kRouteOneCta;
    need(!lists || work_bytes >= moe_route_work_bytes(T, c.n_experts), "work must hold moe_route_work_bytes bytes");
    need_device({{logits_dev, "logits", size}, {bias_dev, "bias", 4, true}, {ids_dev, "ids", 4}, {w_dev, "w", 4}, {offsets_dev, "offsets", 4, true},
                 {inv_dev, "inv", 4, true}, {lists ? work_dev : nullptr, "work", 4, !lists}});
    RouteArgs a{logits_dev, stride ? stride : c.n_experts, bias_dev, T, c.n_experts, c.n_used, G, c.n_groups_used, c.n_experts / G,
                c.score == MOE_SCORE_SIGMOID, c.no_renorm == 0, c.scale == 0.0f ? 1.0f : c.scale, ids_dev, w_dev, offsets_dev, inv_dev,
                lists ? (uint32_t *)work_dev : nullptr};
    int device = 0;
    CUDA_OK(cudaGetDevice(&device));
    if (c.logits_type == MOE_TYPE_F32)
      launch_route<float>(a, device, st);
    else if (c.logits_type == MOE_TYPE_F16)
      launch_route<__half>(a, device, st);
    else
      launch_route<__nv_bfloat16>(a, device, st);
  });
}

}  // extern "C"
