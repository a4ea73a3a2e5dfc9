// Routing of a step's logits without a layer: softmax or sigmoid scores, a bias that chooses but does not weigh, groups of
// experts, the top n_used, and the lists of expert order (moe_route_logits_device).
//
// A warp takes a row; lane l holds experts l, l + 32, .... Keys (score + bias) are first worked out in f32 with the fast exponential and
// reciprocal. A bound that n_used of the lanes' own largest keys reach, found by halving between the least and the largest of them, is one that
// n_used keys reach: the few keys not under it are gathered, one a lane, and each finds its rank by looking at the others. That decides the
// row when every two neighbours among the first n_used + 1 are further apart than the f32 keys' error (key_error): the order is then that of the
// exact keys. Else (a row in some 600 for a bias and 512 experts) the candidates' own keys are worked out in f64, or, where keys that are no
// candidates may come near them, where groups lie that near or ties leave more than 32 keys, the whole row's. Without bias and groups the
// scores' order is the logits' own, which are exact. Renormalised weights come from the chosen logits alone, by the accurate exponential, relative to
// the largest of them, so that they neither overflow nor vanish together; a softmax's that are not, from them and the row's sum of accurate
// exponentials, in f64.
//
// What bounds it: instructions. 32,768 rows of 512 with a bias take 43 us, lists included, 11 of them the bytes at HBM's rate; the rest is a row's
// warp instructions. A warp-wide maximum for each of the first n_used + 1 took 270 us.
//
// The lists: rows are counted by chunks of 32, an expert's rows of a chunk a bit each of a word in shared memory, so that a row's place
// among them is a population count. A scan over the chunks' counts and a pass over the assignments follow; short steps are one cluster's.
#include <cooperative_groups.h>
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
constexpr uint32_t kRouteChunk = 32;       // rows whose experts are counted together
constexpr uint32_t kRouteWarps = 8;        // of a CTA
constexpr uint32_t kRouteShort = 64;       // rows that one cluster of eight CTAs routes and lists by itself, a warp a row
constexpr uint32_t kRoutePlaces = 512;     // assignments a CTA of the last pass takes
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
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }

// Arithmetic of the keys by type. f32: the fast forms, whose errors key_error bounds. f64: what decides.
__device__ __forceinline__ float key_exp(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ double key_exp(double x) { return exp(x); }
template <class T>
__device__ __forceinline__ T minus_inf() {
  return (T)(-INFINITY);
}
__device__ __forceinline__ float sigmoid_key(float l) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + key_exp(-l)));
  return r;
}
__device__ __forceinline__ double sigmoid_key(double l) {
  const double e = exp(l < 0 ? l : -l);  // at most 1
  return (l < 0 ? e : 1.0) / (1.0 + e);
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

// What the f32 score of any of a row's experts may be off by. By PTX's bounds the approximate power of two is within 2^-22 of itself and the
// reciprocal within 2^-23; the exponent x log2(e) is rounded twice, by 2^-23 |x| in all, and l - largest once more. A sigmoid s = 1 / (1 + e)
// moves by s (1 - s) times e's relative error, (1 + |l|) 2^-22 at most, and s (1 - s) (1 + |l|) < 0.5: 2^-20 covers it, the reciprocal and the sum. A softmax
// score e^-d / sum is within (4 + d) 2^-22 of itself, so within 2^-20 of the largest score; and its sum, the mean of (4 + d) over 512
// experts by their e^-d being 8 at most, within 2^-19, and 20 roundings of its own, 2^-19 again at most. The sum's error is all scores' alike, and so
// counts once in the difference of two; so does its reciprocal's rounding, while the products with it are rounded each, 3 x 2^-24 in all. 2 x 2^-20 + 2 x 2^-19
// + 3 x 2^-24 is 6.2 x 2^-20; 2^-18 of the largest score a key is 8 x 2^-20 for two.
__device__ __forceinline__ float key_error(bool sigmoid, float largest_score) { return sigmoid ? 9.5367432e-7f : 3.8146973e-6f * largest_score; }

// Groups, on the warp's E keys in shared memory: each ranked by the sum of its two best; the keys of all but the best a.used become
// -infinity. Returns whether the choice is sure: always for f64; for f32 when the sums of the last group that stays and the first
// that goes are further apart than off, what two of them may be off by, and no group is left out for a sum below f32's range (of keys that a bias
// near the type's lowest value makes), which f64 has room for.
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
    if (best == kNone) {
      sure = !check || !__any_sync(0xffffffffu, two > none && !(one + two > none));
      break;
    }
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

// The row where f32 leaves it open: keys in shared memory, few registers, as it is rare. In f64; without a bias the order, or that within the groups
// that stay, is the logits' own, which scores that vanish or come to 1 would lose. Lane j < k returns the j-th expert.
template <class L>
__device__ __noinline__ uint32_t choose_f64(const RouteArgs &a, uint64_t t, uint32_t lane, float largest, double *sk) {
  const bool scored = a.bias || a.G > 1;
  double sum = 0;
  for (uint32_t e = lane; e < a.E; e += 32) {
    const float l = logit_of<L>(a, t, e);
    sk[e] = l == -INFINITY || !scored ? l : a.sigmoid ? sigmoid_key((double)l) : softmax_part<double>(l, largest);
    if (l > -INFINITY) sum += sk[e];
  }
  if (scored) {
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    for (uint32_t e = lane; e < a.E; e += 32) {
      if (!a.sigmoid) sk[e] /= sum;  // -infinity stays
      if (a.bias && sk[e] > -INFINITY) sk[e] += a.bias[e];
    }
  }
  __syncwarp();
  if (a.G > 1) {
    keep_groups<double>(sk, a, lane, false, 0.0f);
    if (!a.bias)
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

// Whether the lane's i-th expert exists: the launch's V is the least that holds E, so the first half's always do.
template <int V>
__device__ __forceinline__ bool exists(const RouteArgs &a, uint32_t lane, int i) {
  return (V > 1 && i < V / 2) || lane + 32 * i < a.E;
}
// The bias of the lane's experts, as every row of the warp takes it: NaN is out like -infinity.
template <int V>
__device__ __forceinline__ void load_bias(const RouteArgs &a, uint32_t lane, float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; i++) {
    bias[i] = a.bias && exists<V>(a, lane, i) ? a.bias[lane + 32 * i] : 0.0f;
    if (!(bias[i] > -INFINITY)) bias[i] = -INFINITY;
  }
}

// Doubles of shared memory a warp has for a row: a key an expert in f64; or, in 32 bits, 32 candidates' keys and experts and, behind them, all keys.
template <int V>
constexpr uint32_t kRouteScratch = 32 * V;

// One row, by a warp, with kRouteScratch<V> doubles of shared memory of its own. Lane j < k returns the j-th expert (kNone: none) after writing ids and w.
template <class L, int V>
__device__ __forceinline__ uint32_t route_row(const RouteArgs &a, uint64_t t, uint32_t lane, const float (&bias)[V], double *sk) {
  float key[V];  // the logits, then the keys
  const L *row = (const L *)a.logits + t * a.stride + lane;
#pragma unroll
  for (int i = 0; i < V; i++) key[i] = exists<V>(a, lane, i) ? (float)row[32 * i] : -INFINITY;
  const bool scored = a.bias || a.G > 1;
  float largest = -INFINITY, score_max = 1.0f;
  if (!a.sigmoid && (scored || !a.renorm)) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      if (!(key[i] > -INFINITY) || bias[i] == -INFINITY) key[i] = -INFINITY;
      largest = fmaxf(largest, key[i]);
    }
    largest = unordered(__reduce_max_sync(0xffffffffu, ordered(largest)));
    float sum = 0.0f;
    if (a.renorm) {
#pragma unroll
      for (int i = 0; i < V; i++) sum += key[i] == -INFINITY ? 0.0f : softmax_part<float>(key[i], largest);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    } else {
      // The weights are divided by this sum: accurate exponentials, whose errors alone are in it. (32,768 rows of 512 take 56 us so, 46 with the fast ones,
      // whose weights were off by more than eight half steps of f32.)
      double exact = 0.0;
#pragma unroll
      for (int i = 0; i < V; i++) exact += key[i] == -INFINITY ? 0.0f : exp_below(key[i], largest);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) exact += __shfl_xor_sync(0xffffffffu, exact, off);
      sum = (float)exact;
    }
    score_max = largest == -INFINITY ? 0.0f : 1.0f / sum;
  }
  const float err = key_error(a.sigmoid, score_max);
  bool sure = true;
  // v[i] becomes the expert's key, -infinity or NaN if it is out. Rows without experts out, by a minimum over the logits, take no look at each.
  auto to_keys = [&](float (&v)[V]) {
    if (a.sigmoid) {
      float low = INFINITY;
#pragma unroll
      for (int i = 0; i < V; i++) asm("min.NaN.f32 %0, %0, %1;" : "+f"(low) : "f"(key[i]));
      if (__any_sync(0xffffffffu, !(low > -INFINITY))) {
#pragma unroll
        for (int i = 0; i < V; i++) key[i] = key[i] > -INFINITY ? key[i] : __uint_as_float(0x7FFFFFFFu);
      }
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = sigmoid_key(key[i]) + bias[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = softmax_part<float>(key[i], largest) * score_max + bias[i] + (key[i] > -INFINITY ? 0.0f : -INFINITY);
    }
  };
  if (a.G > 1) {
    float *fk = (float *)sk, v[V], top = 0.0f;
    to_keys(v);
#pragma unroll
    for (int i = 0; i < V; i++) {
      const bool out = !(v[i] > -INFINITY);
      if (exists<V>(a, lane, i)) fk[lane + 32 * i] = out ? -INFINITY : v[i];
      top = fmaxf(top, out ? 0.0f : fabsf(v[i]));
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    __syncwarp();
    // Two sums of two keys, each with its own rounding, and theirs.
    sure = keep_groups<float>(fk, a, lane, true, 4 * err + 4.7683716e-7f * top);
    // Without a bias the order within the groups that stay is the logits' own.
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float w = exists<V>(a, lane, i) ? fk[lane + 32 * i] : -INFINITY;
      key[i] = w == -INFINITY ? -INFINITY : a.bias ? w : key[i];
    }
    __syncwarp();
  } else if (a.bias) {
    to_keys(key);
  }
  // least: need keys at least are not under it. It begins as the least of the lanes' largest keys, where need of them are finite, and rises to
  // the middle between it and the largest as long as need of them reach that; ten steps at most, fewer once few more than need do.
  const uint32_t need = a.bias ? a.k + 1 : a.k;  // with a bias the first key left out is looked at too
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; i++) best = fmaxf(best, key[i]);  // NaN loses
  constexpr float kLowest = -3.402823466e38f;
  float least = kLowest, most = unordered(__reduce_max_sync(0xffffffffu, ordered(best)));
  uint32_t reach = __popc(__ballot_sync(0xffffffffu, best >= kLowest));
  if (reach > need) {
    least = unordered(__reduce_min_sync(0xffffffffu, best >= kLowest ? ordered(best) : 0xFFFFFFFFu));
    for (int step = 0; step < 10 && reach > need + 2; step++) {
      const float mid = 0.5f * least + 0.5f * most;
      const uint32_t c = __popc(__ballot_sync(0xffffffffu, best >= mid));
      if (c >= need)
        least = mid, reach = c;
      else
        most = mid;
    }
  }
  // The keys from there on, a lane each.
  uint32_t bits = 0;  // bit i: the lane's i-th is one
#pragma unroll
  for (int i = 0; i < V; i++) bits |= key[i] >= least ? 1u << i : 0u;
  const uint32_t mine = __popc(bits);
  uint32_t upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= (uint32_t)off) upto += o;
  }
  const uint32_t n = __shfl_sync(0xffffffffu, upto, 31);
  uint32_t id = kNone;
  if (n > 32) sure = false;
  if (sure && n > 0) {
    float *found = (float *)sk;                // the keys, and behind them
    uint32_t *expert = (uint32_t *)sk + 32;    // their experts
    uint32_t put = upto - mine;
    // Through shared memory a lane takes its few by their numbers, where registers would want a branch a key.
    if constexpr (V == 1) {
      if (bits) found[put] = key[0], expert[put] = lane;
    } else {
      float *all = (float *)sk + 64 + lane;
#pragma unroll
      for (int i = 0; i < V; i++) all[32 * i] = key[i];
      for (uint32_t left = bits; left; left &= left - 1) {
        const uint32_t i = 32 * (__ffs(left) - 1);
        found[put] = all[i], expert[put++] = lane + i;
      }
    }
    if (lane >= n) found[lane] = -INFINITY;
    __syncwarp();
    const float own = found[lane];
    const uint32_t own_e = expert[lane];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; j += 4) {
      const float4 o = *(const float4 *)(found + j);
      rank += (o.x > own ? 1u : 0u) + (o.y > own ? 1u : 0u) + (o.z > own ? 1u : 0u) + (o.w > own ? 1u : 0u);
    }
    // Without ties the ranks are 0 .. n - 1. With them, a lane's equals of lower experts come before it too.
    if (__reduce_add_sync(0xffffffffu, lane < n ? rank : 0u) != n * (n - 1) / 2)
      for (uint32_t j = 0; j < n; j++) rank += found[j] == own && expert[j] < own_e ? 1u : 0u;
    __syncwarp();
    if (lane < n) found[rank] = own, expert[rank] = own_e;
    __syncwarp();
    const float here = found[lane], next = found[min(lane + 1, 31u)];
    const uint32_t e = expert[lane];
    __syncwarp();
    if (lane < a.k && lane < n) id = e;
    // With a bias no two neighbours may lie within what their scores and their sums' roundings may be off by (rounding keeps an order, so
    // neighbours are all that has to be looked at). Without one the keys are the logits, as they are.
    if (a.bias) {
      const float off = 2 * err + 2.3841858e-7f * fmaxf(fabsf(here), fabsf(next));
      const bool open = lane < a.k && lane + 1 < n && !(here - next > off);
      sure = !__any_sync(0xffffffffu, open);
      // Sigmoids of the candidates alone in f64, a lane each, where no other key can come near the last one taken.
      const float kth = __shfl_sync(0xffffffffu, here, a.k - 1);
      if (!sure && a.sigmoid && n >= need && kth - least > 2 * err + 2.3841858e-7f * fmaxf(fabsf(kth), fabsf(least))) {
        const double v = lane < n ? sigmoid_key((double)logit_of<L>(a, t, e)) + a.bias[e] : -INFINITY;
        rank = 0;
        for (uint32_t j = 0; j < n; j++) {
          const double o = __shfl_sync(0xffffffffu, v, j);
          const uint32_t oe = __shfl_sync(0xffffffffu, e, j);
          rank += o > v || (o == v && oe < e) ? 1u : 0u;
        }
        uint32_t *place = (uint32_t *)sk;
        if (lane < n) place[rank] = e;
        __syncwarp();
        if (lane < a.k) id = place[lane];
        __syncwarp();
        sure = true;
      }
    }
  }
  if (!sure) {
    float l = -INFINITY;
    for (uint32_t e = lane; e < a.E; e += 32) l = fmaxf(l, logit_of<L>(a, t, e));
    id = choose_f64<L>(a, t, lane, unordered(__reduce_max_sync(0xffffffffu, ordered(l))), sk);
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
        s = __fdividef(1.0f, 1.0f + expf(-lj));
      else
        s = __fdividef(exp_below(lj, c), 1.0f + expf(lj));
    }
    float sum = s;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (id != kNone) s = __fdividef(s, sum);  // the largest's own e^0 is in the sum
  } else if (id != kNone) {
    const float ex = a.sigmoid ? expf(-fabsf(lj)) : exp_below(lj, largest);
    s = !a.sigmoid ? ex * score_max : __fdividef(lj < 0.0f ? ex : 1.0f, 1.0f + ex);
  }
  if (lane < a.k) {
    a.ids[t * a.k + lane] = (int32_t)id;
    a.w[t * a.k + lane] = s * a.scale;
  }
  return id;
}

// A chunk of rows by a CTA. With lists, each expert's count of the chunk's rows, and every assignment's place among its expert's rows there.
template <class L, int V>
__global__ void __launch_bounds__(32 * kRouteWarps, 4) k_route_rows(const RouteArgs a) {
  __shared__ __align__(16) double sk[kRouteWarps][kRouteScratch<V>];
  __shared__ uint32_t rows_of[32 * V];  // a bit a row
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (a.work) {
    for (uint32_t i = threadIdx.x; i < a.E; i += 32 * kRouteWarps) rows_of[i] = 0;
    __syncthreads();
  }
  float bias[V];
  load_bias(a, lane, bias);
  const uint32_t t0 = blockIdx.x * kRouteChunk, t1 = min(a.T, t0 + kRouteChunk);
  for (uint32_t t = t0 + warp; t < t1; t += kRouteWarps) {
    const uint32_t id = route_row<L, V>(a, t, lane, bias, sk[warp]);
    if (a.work && id != kNone) atomicOr(&rows_of[id], 1u << (t - t0));
  }
  if (!a.work) return;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.E; i += 32 * kRouteWarps) a.work[(uint64_t)blockIdx.x * a.E + i] = __popc(rows_of[i]);
  const uint64_t a0 = (uint64_t)t0 * a.k;
  for (uint32_t i = threadIdx.x; i < (t1 - t0) * a.k; i += 32 * kRouteWarps) {
    const uint32_t e = (uint32_t)a.ids[a0 + i];  // this CTA's own writes, before the barrier
    a.inv[a0 + i] = e < a.E ? (int32_t)__popc(rows_of[e] & ((1u << i / a.k) - 1)) : -1;
  }
}

// The chunks' counts become each expert's rows before the chunk; the totals come after the last chunk's. A CTA takes 8 experts (a sector of a
// chunk's counts), eight threads a 128th of the chunks, eight counts each on their way at once.
__global__ void __launch_bounds__(1024) k_route_scan(uint32_t *work, uint32_t chunks, uint32_t E) {
  __shared__ uint32_t part[32][8];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, e = blockIdx.x * 8 + lane % 8;
  const uint32_t per = (chunks + 127) / 128, c0 = min(chunks, (warp * 4 + lane / 8) * per), c1 = e < E ? min(chunks, c0 + per) : c0;
  uint32_t *at = work + e, v[8];
  auto load = [&](uint32_t c) {
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) v[j] = c + j < c1 ? at[(uint64_t)(c + j) * E] : 0;
  };
  uint32_t sum = 0;
  for (uint32_t c = c0; c < c1; c += 8) {
    load(c);
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) sum += v[j];
  }
  // Before this thread's chunks: those of the warp's threads 8, 16, 24 lanes down, and of the warps before.
  uint32_t run = 0, all = sum;
  __syncwarp();
#pragma unroll
  for (uint32_t d = 8; d < 32; d += 8) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) run += o;
  }
  all += run;
  if (lane >= 24) part[warp][lane - 24] = all;
  __syncthreads();
  for (uint32_t i = 0; i < warp; i++) run += part[i][lane % 8];
  for (uint32_t c = c0; c < c1; c += 8) {
    if (per > 8) load(c);  // else they are here still
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) {
      if (c + j < c1) at[(uint64_t)(c + j) * E] = run;
      run += v[j];
    }
  }
  if (threadIdx.x >= 1016 && e < E) at[(uint64_t)chunks * E] = run;
}

// Exclusive sums of E <= 512 counts, thread i's of experts 2 i and 2 i + 1, by a block of 8 warps; s: 8 words.
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t pair, uint32_t *s) {
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t v = pair;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= (uint32_t)off) v += o;
  }
  if (lane == 31) s[warp] = v;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t i = 0; i < warp; i++) before += s[i];
  return before + v - pair;
}

// Each assignment's row: its expert's first, the expert's rows of earlier chunks, and its place in its own chunk, which inv holds.
// CTA 0 leaves the offsets.
__global__ void __launch_bounds__(256) k_route_places(const RouteArgs a, uint32_t chunks) {
  __shared__ uint32_t s_scan[8], s_first[kRouteMaxExperts];
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t e = 2 * threadIdx.x;
  const uint32_t *total = a.work + (uint64_t)chunks * a.E;
  const uint32_t n0 = e < a.E ? total[e] : 0, n1 = e + 1 < a.E ? total[e + 1] : 0, first = exclusive_sum(n0 + n1, s_scan);
  s_first[e] = first, s_first[e + 1] = first + n0;
  if (blockIdx.x == 0) {
    if (e < a.E) a.offsets[e] = (int32_t)first;
    if (e + 1 < a.E) a.offsets[e + 1] = (int32_t)(first + n0);
    if (e == a.E - 1 || e + 1 == a.E - 1) a.offsets[a.E] = (int32_t)(first + n0 + n1);
  }
  __syncthreads();
  const uint64_t A = (uint64_t)a.T * a.k, a0 = (uint64_t)blockIdx.x * kRoutePlaces;
  const uint32_t per = kRouteChunk * a.k;  // assignments of a chunk
#pragma unroll
  for (uint32_t j = 0; j < kRoutePlaces / 256; j++) {
    const uint64_t i = a0 + j * 256 + threadIdx.x;
    if (i >= A) break;
    const uint32_t id = (uint32_t)a.ids[i];
    if (id < a.E) a.inv[i] += (int32_t)(s_first[id] + a.work[(i / per) * a.E + id]);
  }
}

// A short step in one launch, a warp a row: a cluster of up to eight CTAs, each with eight rows, which read one another's counts. (One CTA of 32 warps
// took 11 us for 37 rows in groups, bound by its SM's issue slots; this takes 6.)
template <class L, int V>
__global__ void __launch_bounds__(32 * kRouteWarps) k_route_short(const RouteArgs a) {
  __shared__ __align__(16) double sk[kRouteWarps][kRouteScratch<V>];
  __shared__ uint32_t s_scan[8], s_first[kRouteMaxExperts];
  __shared__ __align__(8) uint32_t rows_of[kRouteMaxExperts];  // a bit a row of this CTA
  __shared__ uint64_t all_rows_of[kRouteMaxExperts];           // a bit a row
  dependents_may_launch(), wait_for_predecessors();
  const uint32_t i = threadIdx.x, warp = i / 32, lane = i % 32, t = blockIdx.x * kRouteWarps + warp;
  rows_of[2 * i] = rows_of[2 * i + 1] = 0;
  __syncthreads();
  uint32_t id = kNone;
  if (t < a.T) {
    float bias[V];
    load_bias(a, lane, bias);
    id = route_row<L, V>(a, t, lane, bias, sk[warp]);
    if (a.offsets && id != kNone) atomicOr(&rows_of[id], 1u << warp);
  }
  if (!a.offsets) return;
  const uint32_t e = 2 * i;
  uint64_t r0 = 0, r1 = 0;
  if (gridDim.x == 1) {  // a CTA alone is launched as no cluster
    __syncthreads();
    r0 = rows_of[e], r1 = rows_of[e + 1];
  } else {
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    for (uint32_t c = 0; c < gridDim.x; c++) {
      const uint2 r = *(const uint2 *)(cluster.map_shared_rank(rows_of, c) + e);
      r0 |= (uint64_t)r.x << kRouteWarps * c, r1 |= (uint64_t)r.y << kRouteWarps * c;
    }
    cluster.sync();  // no CTA leaves while another reads its counts
  }
  all_rows_of[e] = r0, all_rows_of[e + 1] = r1;
  const uint32_t n0 = __popcll(r0), n1 = __popcll(r1), first = exclusive_sum(n0 + n1, s_scan);
  s_first[e] = first, s_first[e + 1] = first + n0;
  if (blockIdx.x == 0) {
    if (e < a.E) a.offsets[e] = (int32_t)first;
    if (e + 1 < a.E) a.offsets[e + 1] = (int32_t)(first + n0);
    if (e == a.E - 1 || e + 1 == a.E - 1) a.offsets[a.E] = (int32_t)(first + n0 + n1);
  }
  __syncthreads();
  if (t < a.T && lane < a.k)
    a.inv[(uint64_t)t * a.k + lane] = id < a.E ? (int32_t)(s_first[id] + __popcll(all_rows_of[id] & ((1ull << t) - 1))) : -1;
}

__global__ void __launch_bounds__(512) k_route_empty(int32_t *offsets, uint32_t n) {
  dependents_may_launch(), wait_for_predecessors();
  for (uint32_t i = threadIdx.x; i < n; i += 512) offsets[i] = 0;
}

template <class L, int V>
void launch_rows(const RouteArgs &a, cudaStream_t st) {
  if (a.T <= kRouteShort) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension, at[1].val.clusterDim = {(a.T + kRouteWarps - 1) / kRouteWarps, 1, 1};
    cfg.gridDim = dim3(at[1].val.clusterDim.x), cfg.blockDim = dim3(32 * kRouteWarps), cfg.stream = st, cfg.attrs = at, cfg.numAttrs = cfg.gridDim.x > 1 ? 2 : 1;
    CUDA_OK(cudaLaunchKernelEx(&cfg, k_route_short<L, V>, a));
    return;
  }
  const uint32_t chunks = (a.T + kRouteChunk - 1) / kRouteChunk;
  CUDA_OK(launch_kernel(true, k_route_rows<L, V>, dim3(chunks), dim3(32 * kRouteWarps), 0, st, a));
  if (!a.offsets) return;
  CUDA_OK(launch_kernel(true, k_route_scan, dim3((a.E + 7) / 8), dim3(1024), 0, st, a.work, chunks, a.E));
  CUDA_OK(launch_kernel(true, k_route_places, dim3((uint32_t)(((uint64_t)a.T * a.k + kRoutePlaces - 1) / kRoutePlaces)), dim3(256), 0, st, a, chunks));
}

template <class L>
void launch_route(const RouteArgs &a, cudaStream_t st) {
  if (a.E <= 32)
    launch_rows<L, 1>(a, st);
  else if (a.E <= 64)
    launch_rows<L, 2>(a, st);
  else if (a.E <= 128)
    launch_rows<L, 4>(a, st);
  else if (a.E <= 256)
    launch_rows<L, 8>(a, st);
  else
    launch_rows<L, 16>(a, st);
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
    const bool lists = offsets_dev && T > kRouteShort;
    need(!lists || work_bytes >= moe_route_work_bytes(T, c.n_experts), "work must hold moe_route_work_bytes bytes");
    need_device({{logits_dev, "logits", size}, {bias_dev, "bias", 4, true}, {ids_dev, "ids", 4}, {w_dev, "w", 4}, {offsets_dev, "offsets", 4, true},
                 {inv_dev, "inv", 4, true}, {lists ? work_dev : nullptr, "work", 4, !lists}});
    RouteArgs a{logits_dev, stride ? stride : c.n_experts, bias_dev, T, c.n_experts, c.n_used, G, c.n_groups_used, c.n_experts / G,
                c.score == MOE_SCORE_SIGMOID, c.no_renorm == 0, c.scale == 0.0f ? 1.0f : c.scale, ids_dev, w_dev, offsets_dev, inv_dev,
                lists ? (uint32_t *)work_dev : nullptr};
    if (c.logits_type == MOE_TYPE_F32)
      launch_route<float>(a, st);
    else if (c.logits_type == MOE_TYPE_F16)
      launch_route<__half>(a, st);
    else
      launch_route<__nv_bfloat16>(a, st);
  });
}

}  // extern "C"
