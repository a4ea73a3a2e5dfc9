// Rows to expert order in their own type, and the gradients of that and of the combine (include/moe_layer.h). Single passes over their data, bound by HBM in long steps:
// a row is read once and written to its places, or its places are read four rows at a time and summed. No sum is by atomics, and each has one order.
// 32,768 rows of 2,048 bf16 values to ten places each 234 us (6.3 TB/s); the combine's gradients of 16,384 such rows 235 (6.3); rows' and weights' gradients of 3,521
// rows of 2,560 f16 values, eight places each, 31.5 (5.2), of 8,192 of 2,048 bf16 57 (5.9), rows' alone 50 (6.0); of 90,000 rows of 64 29 (3.9). 13 rows of 2,560 f32
// values to eight places each 1.8 us.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "mx4.cuh"
#include "ops_common.h"

namespace moe {
namespace {

constexpr uint32_t kRowsMaxUsed = 16;
constexpr uint32_t kThreads = 256;
constexpr uint32_t kLongStep = 1024;  // rows
constexpr uint32_t kFewThreads = 148 * 512;  // a step's, at least

// How a step's rows are dealt to a CTA of 256 threads: 2^log2 neighbouring threads a row; of its octets, groups of eight values, thread i takes i,
// i + 2^log2 and so on; with several CTAs a row (grid.y) they take turns.
struct StepRows {
  uint32_t T, log2, octets;
  __device__ uint64_t row() const { return (uint64_t)blockIdx.x * (kThreads >> log2) + (threadIdx.x >> log2); }
  __device__ uint32_t first() const { return (threadIdx.x & ((1u << log2) - 1)) + (blockIdx.y << log2); }
  __device__ uint32_t step() const { return gridDim.y << log2; }
};

// Here the map's octets are pieces of 16 bytes, so that neighbouring threads store neighbouring ones (of f32 rows two pieces a thread, every other one at a time, took 74 us
// of 7,787 rows of 768, eleven places each, where this takes 47). U of them at a time, whose loads are on their way together.
template <class X, uint32_t U>
__global__ void __launch_bounds__(kThreads) k_sort_rows(const X *x, uint64_t stride, const StepRows map, const int32_t *inv, const float *w, uint32_t n_used, uint32_t R,
                                                        X *xs) {
  dependents_may_launch(), wait_for_predecessors();
  constexpr uint32_t V = 16 / sizeof(X);
  const uint64_t t = map.row(), D = (uint64_t)V * map.octets;
  if (t >= map.T) return;
  for (uint32_t o = map.first(); o < map.octets; o += U * map.step()) {
    uint4 raw[U];
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
      if (o + u * map.step() < map.octets) raw[u] = *(const uint4 *)(x + t * stride + V * (o + u * map.step()));
#pragma unroll 4
    for (uint32_t j = 0; j < n_used; j++) {
      const uint32_t r = (uint32_t)inv[t * n_used + j];
      if (r >= R) continue;
      const float f = w ? w[t * n_used + j] : 1.0f;
#pragma unroll
      for (uint32_t u = 0; u < U; u++) {
        if (o + u * map.step() >= map.octets) break;
        X *to = xs + r * D + V * (o + u * map.step());
        if (!w) {
          *(uint4 *)to = raw[u];
        } else if constexpr (V == 4) {
          const float4 v = *(const float4 *)&raw[u];
          *(float4 *)to = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        } else {
          float v[8];
          load8((const X *)&raw[u], v);
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] *= f;
          store8(to, v);
        }
      }
    }
  }
}

// Up to four rows' octets as they were loaded.
template <class X>
struct FourRows {
  uint4 raw[4][sizeof(X) / 2];
  uint32_t r[4];
  // Rows inv[j0] .. inv[j0 + 3] of those there are, those of R alone.
  __device__ void load(const X *rows, uint64_t D, uint32_t c, const int32_t *inv, uint32_t j0, uint32_t n, uint32_t R, bool wanted = true) {
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) r[j] = j0 + j < n ? (uint32_t)inv[j0 + j] : 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
#pragma unroll
      for (uint32_t i = 0; i < sizeof(X) / 2; i++)
        if (wanted && r[j] < R) raw[j][i] = ((const uint4 *)(rows + r[j] * D + c))[i];
  }
  __device__ void values(uint32_t j, float *v) const { load8((const X *)raw[j], v); }
};

// The sums of N = 4 Q numbers a thread over a row's 2^log2 threads, n of them to out. The CTA's threads come here together. (Numbers, not lanes, are halved by the
// first exchanges, each lane keeping those whose index has its bits: 16 exchanges a warp for 16 numbers instead of 80.)
template <uint32_t Q>
__device__ __forceinline__ void row_sums(float (&of)[4 * Q], uint32_t log2, float (*part)[kRowsMaxUsed], bool in, uint32_t n, float *out) {
  constexpr uint32_t N = Q == 1 ? 4 : Q == 2 ? 8 : 16;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float d[N];
#pragma unroll
  for (uint32_t j = 0; j < N; j++) d[j] = j < 4 * Q ? of[j] : 0.0f;
  if (log2 >= 5) {
    uint32_t mine = 0;  // the number whose sum the lane comes to hold
#pragma unroll
    for (uint32_t h = N / 2, bit = 16; h; h /= 2, bit /= 2) {
#pragma unroll
      for (uint32_t i = 0; i < h; i++) {
        const float keep = lane & bit ? d[i + h] : d[i], give = lane & bit ? d[i] : d[i + h];
        d[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
      }
      mine += lane & bit ? h : 0;
    }
#pragma unroll
    for (uint32_t bit = 16 / N; bit; bit /= 2) d[0] += __shfl_xor_sync(0xffffffffu, d[0], bit);
    const bool first = lane % (32 / N) == 0;
    if (log2 == 5) {
      if (in && first && mine < n) out[mine] = d[0];
      return;
    }
    if (first) part[warp][mine] = d[0];
    __syncthreads();
    const uint32_t i = threadIdx.x & ((1u << log2) - 1), each = 1u << (log2 - 5);
    if (in && i < n) {
      float s = 0.0f;
      for (uint32_t k = 0; k < each; k++) s += part[(warp & ~(each - 1)) + k][i];
      out[i] = s;
    }
    return;
  }
  const uint32_t i = lane & ((1u << log2) - 1);
#pragma unroll
  for (uint32_t j = 0; j < 4 * Q; j++) {
    for (uint32_t off = (1u << log2) / 2; off; off /= 2) d[j] += __shfl_xor_sync(0xffffffffu, d[j], off);
    if (in && i == 0 && j < n) out[j] = d[j];
  }
}

// CTAs an SM of the gradients' kernels, by the registers that four rows' octets as they were loaded, their sums and the row's own values take: 8,192 rows of 2,048 bf16
// values, dx and dw, 63 us with four, 71 with three, 75 with five (which spill); 4,096 of 4,096 f32 values 101 with three, 132 with two.
template <class X>
constexpr uint32_t grad_ctas() {
  return sizeof(X) == 4 ? 3 : 4;
}

// dx[t] = (add[t] +) sum_j (w[t][j]) dxs[inv[t][j]], and where dw is wanted dw[t][j] = <x[t], dxs[inv[t][j]]>. Q: fours of results a row has.
template <class X, bool DW, uint32_t Q>
__global__ void __launch_bounds__(kThreads, grad_ctas<X>()) k_sort_rows_grad(const X *dxs, const StepRows map, uint32_t R, const int32_t *inv, const float *w, const X *x,
                                                                             uint64_t stride, uint32_t n_used, const X *add, X *dx, float *dw) {
  __shared__ float part[DW ? kThreads / 32 : 1][kRowsMaxUsed];
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t t = map.row(), D = 8ull * map.octets;
  const bool in = t < map.T;
  float dot[DW ? 4 * Q : 1] = {};
  if (in) {
    inv += t * n_used, w += w ? t * n_used : 0;
    for (uint32_t o = map.first(); o < map.octets; o += map.step()) {
      float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, xv[8];
      if constexpr (DW) load8(x + t * stride + 8 * o, xv);
#pragma unroll
      for (uint32_t j0 = 0; j0 < 4 * Q; j0 += 4) {
        FourRows<X> rows;
        rows.load(dxs, D, 8 * o, inv, j0, n_used, R);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          if (rows.r[j] >= R) continue;
          const float f = w ? w[j0 + j] : 1.0f;
          float v[8];
          rows.values(j, v);
#pragma unroll
          for (int i = 0; i < 8; i++) acc[i] = fmaf(f, v[i], acc[i]);
          if constexpr (DW)
#pragma unroll
            for (int i = 0; i < 8; i++) dot[j0 + j] = fmaf(xv[i], v[i], dot[j0 + j]);
        }
      }
      if (dx) {
        if (add) {
          float v[8];
          load8(add + t * D + 8 * o, v);
#pragma unroll
          for (int i = 0; i < 8; i++) acc[i] += v[i];
        }
        store8(dx + t * D + 8 * o, acc);
      }
    }
  }
  if constexpr (DW) row_sums<Q>(dot, map.log2, part, in, n_used, dw + t * n_used);
}

// dy[inv[t][j]] = w[t][j] dout[t], dw[t][j] = <dout[t], y[inv[t][j]]>. dy may be y: a thread has read what it writes over.
template <class G, class Y, uint32_t Q>
__global__ void __launch_bounds__(kThreads, grad_ctas<Y>()) k_combine_rows_grad(const G *dout, const Y *y, const StepRows map, uint32_t R, const int32_t *inv, const float *w,
                                                                                uint32_t n_used, Y *dy, float *dw) {
  __shared__ float part[kThreads / 32][kRowsMaxUsed];
  dependents_may_launch(), wait_for_predecessors();
  const uint64_t t = map.row(), D = 8ull * map.octets;
  const bool in = t < map.T;
  float dot[4 * Q] = {};
  if (in) {
    inv += t * n_used, w += w ? t * n_used : 0;
    for (uint32_t o = map.first(); o < map.octets; o += map.step()) {
      float g[8];
      load8(dout + t * D + 8 * o, g);
#pragma unroll
      for (uint32_t j0 = 0; j0 < 4 * Q; j0 += 4) {
        FourRows<Y> rows;
        rows.load(y, D, 8 * o, inv, j0, n_used, R, dw);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          if (rows.r[j] >= R) continue;
          if (dy) {
            const float f = w[j0 + j];
            float u[8];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = f * g[i];
            store8(dy + rows.r[j] * D + 8 * o, u);
          }
          if (dw) {
            float v[8];
            rows.values(j, v);
#pragma unroll
            for (int i = 0; i < 8; i++) dot[j0 + j] = fmaf(g[i], v[i], dot[j0 + j]);
          }
        }
      }
    }
  }
  if (dw) row_sums<Q>(dot, map.log2, part, in, n_used, dw + t * n_used);
}

// Calls f with the fours of results a row has, as a type.
template <class F>
void with_fours(uint32_t n_used, F &&f) {
  using std::integral_constant;
  if (n_used <= 4)
    f(integral_constant<uint32_t, 1>{});
  else if (n_used <= 8)
    f(integral_constant<uint32_t, 2>{});
  else if (n_used <= 12)
    f(integral_constant<uint32_t, 3>{});
  else
    f(integral_constant<uint32_t, 4>{});
}

// Calls f with the map for a step's rows, and its grid. Rows of more than 32 octets get up to a CTA of threads. least_log2 and most_log2 are for long steps: as many
// threads a row, within them, as leave fewer than an eighth of them idle in a row's last round, but enough to fill the GPU (1,030 rows of 1,320, twelve places: the
// combine's gradients 17 us so, 29 with a warp a row). What only reads rows does best with a warp a row, which meets at no barrier (8,192 rows of 2,048 bf16 values, eight
// places each, dx and dw: 57 us, 59 with 64 threads a row, 62 with 256; of 1,536 44, 46 and 56); the combine's gradients, which write them too, with as many threads as
// fit (16,384 of 2,048, ten places: 232 us with 256, 244 with 32; 4,096 of 2,880, six places: 58 with 64, 61 with 256, 64 with 32); sorting with 256 whatever is
// idle (3,163 of 1,776 bf16 values, thirteen places: 28.6 us, 35.6 with 32). whole: a row is one CTA's; else a short step's rows are up to 16 CTAs'.
template <class F>
void with_step_rows(uint32_t T, uint32_t n_embd, uint32_t least_log2, uint32_t most_log2, bool whole, F &&f) {
  StepRows map{T, 0, n_embd / 8};
  while (map.log2 < 8 && (1u << map.log2) < map.octets) map.log2++;
  if (T >= kLongStep && map.log2 > 5) {
    auto slots = [&](uint32_t log2) { return (uint64_t)((map.octets + (1u << log2) - 1) >> log2) << log2; };
    uint32_t log2 = std::min(most_log2, map.log2);
    while (log2 > least_log2 && slots(log2) * 8 > map.octets * 9ull) log2--;
    while (log2 < map.log2 && (uint64_t)T << log2 < kFewThreads) log2++;
    map.log2 = log2;
  }
  const uint32_t rows = kThreads >> map.log2, rounds = (map.octets + (1u << map.log2) - 1) >> map.log2;
  f(map, dim3((T + rows - 1) / rows, whole || T >= kLongStep ? 1 : std::min(rounds, 16u)));
}

void need_step(uint32_t T, uint32_t R, uint32_t n_used, uint32_t n_embd) {
  need(n_used >= 1 && n_used <= kRowsMaxUsed, "n_used must be 1 .. 16");
  need(n_embd >= 8 && n_embd % 8 == 0 && n_embd <= 1u << 24, "n_embd must be a multiple of 8, at most 2^24");
  need(T < 1u << 31 && R < 1u << 31, "T and R must be below 2^31");
}

void need_stride(uint64_t stride, uint32_t n_embd, uint32_t size) {
  need(stride == 0 || (stride >= n_embd && stride < 1ull << 32 && stride * size % 16 == 0), "stride must be 0, or n_embd at least with rows 16-byte aligned");
}

// Calls f with a null pointer of the type's element.
template <class F>
void with_type(uint32_t type, F &&f) {
  if (type == MOE_TYPE_F32)
    f((float *)nullptr);
  else if (type == MOE_TYPE_F16)
    f((__half *)nullptr);
  else
    f((__nv_bfloat16 *)nullptr);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

MOE_API moe_status moe_sort_rows_device(const void *x_dev, uint32_t type, uint64_t stride, uint32_t T, uint32_t n_used, uint32_t n_embd, const int32_t *inv_dev,
                                        const float *w_dev, uint32_t R, void *xs_dev, void *stream) {
  return ops_call([&] {
    const uint32_t size = row_type_bytes(type);
    need(size != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_step(T, R, n_used, n_embd);
    need_stride(stride, n_embd, size);
    if (T == 0 || R == 0) return;
    need_device({{x_dev, "x", 16}, {inv_dev, "inv", 4}, {w_dev, "w", 4, true}, {xs_dev, "xs", 16}});
    with_step_rows(T, n_embd / 2 * size, 8, 8, false, [&](StepRows map, dim3 grid) {
      with_type(type, [&](auto *of) {
        using X = std::remove_pointer_t<decltype(of)>;
        // Pieces a thread has of a row, up to four at a time (13,516 rows of 3,768 weighted bf16 values, three places each, 70 us, one at a time 79; 32,768 of 2,048, one
        // place, 45 and 50).
        const uint32_t mine = (map.octets + (grid.y << map.log2) - 1) / (grid.y << map.log2);
        const auto kernel = mine == 1 ? k_sort_rows<X, 1> : mine == 2 ? k_sort_rows<X, 2> : k_sort_rows<X, 4>;
        CUDA_OK(launch_kernel(true, kernel, grid, dim3(kThreads), 0, (cudaStream_t)stream, (const X *)x_dev, stride ? stride : n_embd, map, inv_dev, w_dev, n_used, R,
                              (X *)xs_dev));
      });
    });
  });
}

MOE_API moe_status moe_sort_rows_grad_device(const void *dxs_dev, uint32_t type, uint32_t R, const int32_t *inv_dev, const float *w_dev, const void *x_dev, uint64_t stride,
                                             uint32_t T, uint32_t n_used, uint32_t n_embd, const void *add_dev, void *dx_dev, float *dw_dev, void *stream) {
  return ops_call([&] {
    const uint32_t size = row_type_bytes(type);
    need(size != 0, "type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_step(T, R, n_used, n_embd);
    need_stride(stride, n_embd, size);
    need(dx_dev || dw_dev, "dx or dw is required");
    need(!dw_dev || x_dev, "x is required for dw");
    need(!add_dev || dx_dev, "dx is required with add");
    if (T == 0) return;
    // With R 0 no row of dxs is read: it may be null then.
    need_device({{dxs_dev, "dxs", 16, R == 0}, {inv_dev, "inv", 4}, {w_dev, "w", 4, true}, {x_dev, "x", 16, true}, {add_dev, "add", 16, true}, {dx_dev, "dx", 16, true},
                 {dw_dev, "dw", 4, true}});
    with_step_rows(T, n_embd, 5, dw_dev ? 5 : 8, dw_dev, [&](StepRows map, dim3 grid) {
      with_type(type, [&](auto *of) {
        using X = std::remove_pointer_t<decltype(of)>;
        with_fours(n_used, [&](auto q) {
          constexpr uint32_t Q = decltype(q)::value;
          const auto kernel = dw_dev ? k_sort_rows_grad<X, true, Q> : k_sort_rows_grad<X, false, Q>;
          CUDA_OK(launch_kernel(true, kernel, grid, dim3(kThreads), 0, (cudaStream_t)stream, (const X *)dxs_dev, map, R, inv_dev, w_dev, (const X *)x_dev,
                                stride ? stride : n_embd, n_used, (const X *)add_dev, (X *)dx_dev, dw_dev));
        });
      });
    });
  });
}

MOE_API moe_status moe_combine_rows_grad_device(const void *dout_dev, uint32_t dout_type, const void *y_dev, uint32_t y_type, uint32_t R, const int32_t *inv_dev,
                                                const float *w_dev, uint32_t T, uint32_t n_used, uint32_t n_embd, void *dy_dev, float *dw_dev, void *stream) {
  return ops_call([&] {
    need(row_type_bytes(dout_type) != 0, "dout_type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need(row_type_bytes(y_type) != 0, "y_type must be MOE_TYPE_F32, MOE_TYPE_F16 or MOE_TYPE_BF16");
    need_step(T, R, n_used, n_embd);
    need(dy_dev || dw_dev, "dy or dw is required");
    need(!dw_dev || y_dev || R == 0, "y is required for dw");
    need(!dy_dev || w_dev, "w is required for dy");
    if (T == 0) return;
    need_device({{dout_dev, "dout", 16}, {y_dev, "y", 16, true}, {inv_dev, "inv", 4}, {w_dev, "w", 4, true}, {dy_dev, "dy", 16, true}, {dw_dev, "dw", 4, true}});
    with_step_rows(T, n_embd, 5, 8, dw_dev, [&](StepRows map, dim3 grid) {
      with_type(dout_type, [&](auto *g) {
        using G = std::remove_pointer_t<decltype(g)>;
        with_type(y_type, [&](auto *of) {
          using Y = std::remove_pointer_t<decltype(of)>;
          with_fours(n_used, [&](auto q) {
            CUDA_OK(launch_kernel(true, k_combine_rows_grad<G, Y, decltype(q)::value>, grid, dim3(kThreads), 0, (cudaStream_t)stream, (const G *)dout_dev,
                                  (const Y *)y_dev, map, R, inv_dev, w_dev, n_used, (Y *)dy_dev, dw_dev));
          });
        });
      });
    });
  });
}

}  // extern "C"
