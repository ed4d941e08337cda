// What the two plans of a ragged extension batch (extend_attention.hip, extend_shared.hip)
// have in common.
#pragma once

#include "extend_common.hpp"

namespace gemma4 {

struct Sum {
  template <class T> __device__ T operator()(T a, T b) const { return a + b; }
};
struct Max {
  template <class T> __device__ T operator()(T a, T b) const { return a > b ? a : b; }
};
// Inclusive prefix of one value per thread over the workgroup; the last
// thread's in `total`.
template <int kWaves, class T, class F>
__device__ __forceinline__ T block_prefix(T x, T &total, T *waves, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const T other = __shfl_up(x, d);
    if (lane >= d) x = f(other, x);
  }
  if (lane == kWave - 1) waves[wave] = x;
  __syncthreads();
  T head = waves[0], all = waves[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    if (w < wave) head = f(head, waves[w]);
    all = f(all, waves[w]);
  }
  total = all;
  __syncthreads();
  return wave > 0 ? f(head, x) : x;
}

constexpr int kPlanShares = 256;
constexpr int kShareTiles = 2;  // least cost worth a workgroup
// Besides its tiles a row block costs the way to its first keys, its queries and its
// rows' end. Where it holds several waves' rows that is 7.8 us at 8 x 256, of 1.3 us a
// tile, and 12 at 1 x 512, of 2.1; where one's, 4.5 and 7.
__device__ __forceinline__ int32_t block_cost(const ExtendGeometry &g, int32_t rows) {
  return rows > g.wave_rows ? 6 : 3;
}

// Host checks of the extension's entry points.
bool extend_sizes_ok(const Gemma4KvCacheConfig &c, int32_t batch, int32_t total_rows);

// The attention by a plan of either kind, after the caller's checks of the plan.
struct ExtendCall {
  gemma4_bf16 *out;
  const gemma4_bf16 *q, *k, *v, *cache_k, *cache_v;
  const int32_t *page_table;
  const void *plan;
  Gemma4KvCacheConfig config;
  int32_t layer, batch, total_rows;
  int64_t q_stride, kv_stride;
  float softmax_scale;
  void *workspace;
  size_t workspace_bytes;
};
inline size_t extend_workspace_bytes(const ExtendPlanLayout &l, const Gemma4KvCacheConfig &c) {
  return (size_t)(extend_odd_offset(l, c.head_dim) + extend_round(l.max_partials * c.num_heads * 16));
}
hipError_t extend_attend(const ExtendCall &call, const ExtendPlanLayout &l, uint32_t magic,
                         int64_t shared_rows, hipStream_t stream);

}  // namespace gemma4
