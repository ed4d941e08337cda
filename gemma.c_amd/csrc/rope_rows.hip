// Preparation of ragged rows, gfx950: RMSNorm and rotary positions of q and k,
// scale-free RMSNorm of v, from a projection's strided rows to packed ones. The
// per-head arithmetic is the reference's (src/gemma4_flash_attention_decode.cu:233-283,
// src/gemma4_rope.cu:8-20); the layouts, the scaled frequencies and the table-free
// angles have no counterpart there.
//
// Workgroup: a row. A lane holds 8 dims of a head, so that a head is half a wave at
// 256 dims and a wave at 512, every access is 16 bytes per lane and the sum of
// squares is a reduction over the head's lanes. The rows are asked for first; while
// they are on their way each pair's angle is worked out once for all heads and put
// into LDS: the turns position * turns[i] in 64 bits (a position has 31 of them and a
// turn's part has to keep 24), the whole ones dropped, the rest in 32. One rounding, of
// the outputs to bf16.
//
// What bounds it: HBM. 2048 rows at 1 x 512 (73 MB) 14.6 us, the rate of a large copy;
// 1348 rows of 12 sequences at 8 x 256 (44 MB) 11.0 us, 82% of it with the launch. All that a
// row needs is asked for before its position is tested: 12.7 us where that came first.
#include "gemma4_device.hpp"
#include "prep_common.hpp"

#include "gemma4_flash_attention.h"

#include <math.h>

namespace gemma4 {
namespace {

struct RopeParams {
  uint16_t *q_out;
  uint16_t *k_out;
  uint16_t *v_out;     // null: no V
  const uint16_t *q;
  const uint16_t *k;
  const uint16_t *v;   // null: V from the raw k
  const uint16_t *q_weight;  // null: q is not normed
  const uint16_t *k_weight;
  const int32_t *position;
  const double *turns;
  int64_t q_stride, kv_stride;
  float amplitude;
  int32_t rotary;
};

constexpr int kMaxPairs = 256;

template <int kDim>
struct RopeShape {
  static constexpr int kHeads = kDim == 256 ? 8 : 1;
  static constexpr int kLanes = kDim / kPackElems;       // of a head
  static constexpr int kItemHeads = kWave / kLanes;      // heads of a wave's pack
  static constexpr int kWaves = kDim == 256 ? 8 : 9;
  static constexpr int kItems = 2;                       // of a wave
};

// Sum over the head's lanes.
template <int kLanes>
__device__ __forceinline__ float head_sum(float x) {
  x += lane_xor<1>(x);
  x += lane_xor<2>(x);
  x += lane_xor<4>(x);
  x += lane_xor<8>(x);
  x = xor_sum<16>(x);
  if constexpr (kLanes == kWave) x = xor_sum<32>(x);
  return x;
}

template <int kDim, bool kInterleaved>
__global__ __launch_bounds__(RopeShape<kDim>::kWaves *kWave) void rope_rows_kernel(RopeParams p) {
  using S = RopeShape<kDim>;
  __shared__ __attribute__((aligned(16))) float s_cos[kMaxPairs], s_sin[kMaxPairs];
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int wave = wave_uniform(t / kWave);
  const int64_t row = blockIdx.x;
  const int32_t position = p.position[row];

  // Items of a row: at 8 x 256 pairs of heads, 8 of q, then 4 of k, then 4 of v, two to
  // a wave; at 1 x 512 heads, two of q to a wave and k with the v made of it to the last.
  const int sub = lane / S::kLanes, d0 = lane % S::kLanes * kPackElems;
  enum Kind { kQ, kK, kV };
  constexpr int kQItems = kQueryHeads / S::kItemHeads;
  auto kind_of = [&](int item) {
    return item < kQItems ? kQ : (S::kHeads == 1 || item < kQItems + S::kHeads / S::kItemHeads ? kK : kV);
  };
  const bool last_wave = S::kHeads == 1 && wave == S::kWaves - 1;
  const int items = last_wave ? 1 : S::kItems;
  uint4 x[S::kItems], raw_v = make_uint4(0, 0, 0, 0);
  auto head_of = [&](int item) {
    const Kind kind = kind_of(item);
    const int first = kind == kQ ? 0 : (kind == kK ? kQItems : kQItems + S::kHeads / S::kItemHeads);
    return (item - first) * S::kItemHeads + sub;
  };
#pragma unroll
  for (int i = 0; i < S::kItems; ++i) {
    const int item = wave * S::kItems + i;
    if (i >= items) break;
    const Kind kind = kind_of(item);
    if (kind == kV && p.v_out == nullptr) continue;
    const uint16_t *from = kind == kQ ? p.q + row * p.q_stride
                                      : (kind == kK || p.v == nullptr ? p.k : p.v) + row * p.kv_stride;
    x[i] = load128(from + head_of(item) * kDim + d0);
    if (S::kHeads == 1 && kind == kK && p.v != nullptr && p.v_out != nullptr)
      raw_v = load128(p.v + row * p.kv_stride + d0);
  }
  // A wave's items are of one kind.
  static_assert(kQItems % S::kItems == 0 && (S::kHeads == 1 || S::kHeads / S::kItemHeads % S::kItems == 0));
  const Kind wave_kind = kind_of(wave * S::kItems);
  const uint16_t *weight = wave_kind == kQ ? p.q_weight : (wave_kind == kK ? p.k_weight : nullptr);
  uint4 raw_w = make_uint4(0, 0, 0, 0);
  if (weight != nullptr) raw_w = load128(weight + d0);
  const int half = p.rotary / 2;
  static_assert(S::kWaves * kWave >= kMaxPairs, "a thread a pair");
  const double per_position = t < half ? p.turns[t] : 0.0;
  // Behind the loads: the row is there, whatever its position.
  if (position < 0) return;
  if (t < half) {
    const double turns = (double)position * per_position;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    s_cos[t] = p.amplitude * c;
    s_sin[t] = p.amplitude * s;
  }
  __syncthreads();

  auto unpacked_scale = [&](const uint4 &raw, float (&y)[kPackElems]) {
    unpack8(raw, y);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPackElems; ++e) sum = fmaf(y[e], y[e], sum);
    return 1.0f / sqrtf(head_sum<S::kLanes>(sum) / (float)kDim + kRmsEps);
  };
  auto store = [&](uint16_t *to, const float (&y)[kPackElems]) {
    store128(to, make_uint4(cvt_pk_bf16(y[0], y[1]), cvt_pk_bf16(y[2], y[3]),
                            cvt_pk_bf16(y[4], y[5]), cvt_pk_bf16(y[6], y[7])));
  };
  auto store_normed = [&](uint16_t *to, const uint4 &raw) {
    float y[kPackElems];
    const float scale = unpacked_scale(raw, y);
#pragma unroll
    for (int e = 0; e < kPackElems; ++e) y[e] *= scale;
    store(to, y);
  };
#pragma unroll
  for (int i = 0; i < S::kItems; ++i) {
    const int item = wave * S::kItems + i;
    if (i >= items) break;
    const Kind kind = kind_of(item);
    const int head = head_of(item);
    if (kind == kV) {
      if (p.v_out != nullptr) store_normed(p.v_out + (row * S::kHeads + head) * kDim + d0, x[i]);
      continue;
    }
    float y[kPackElems];
    if (weight != nullptr) {
      const float scale = unpacked_scale(x[i], y);
      float w[kPackElems];
      unpack8(raw_w, w);
#pragma unroll
      for (int e = 0; e < kPackElems; ++e) y[e] = y[e] * scale * w[e];
    } else {
      unpack8(x[i], y);
    }
    if constexpr (kInterleaved) {
      if (d0 < p.rotary) {
#pragma unroll
        for (int e = 0; e < kPackElems; e += 2) {
          const float c = s_cos[(d0 + e) / 2], s = s_sin[(d0 + e) / 2];
          const float a = y[e], b = y[e + 1];
          y[e] = fmaf(a, c, -b * s);
          y[e + 1] = fmaf(a, s, b * c);
        }
      }
    } else {
      // The pair's other dim sits rotary / 16 lanes on or back.
      const bool low = d0 < half;
      const int partner = lane + (low ? half / kPackElems : -(half / kPackElems));
      float other[kPackElems];
#pragma unroll
      for (int e = 0; e < kPackElems; ++e) other[e] = __shfl(y[e], partner & (kWave - 1));
      if (d0 < p.rotary) {
        const int pair = low ? d0 : d0 - half;
        const float sign = low ? -1.0f : 1.0f;
#pragma unroll
        for (int e = 0; e < kPackElems; ++e)
          y[e] = fmaf(sign * other[e], s_sin[pair + e], y[e] * s_cos[pair + e]);
      }
    }
    if (kind == kQ) {
      store(p.q_out + (row * kQueryHeads + head) * kDim + d0, y);
    } else {
      store(p.k_out + (row * S::kHeads + head) * kDim + d0, y);
      if (S::kHeads == 1 && p.v_out != nullptr)
        store_normed(p.v_out + row * kDim + d0, p.v != nullptr ? raw_v : x[i]);
    }
  }
}

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int kDim>
void launch_rope(const RopeParams &p, int32_t rows, bool interleaved, hipStream_t stream) {
  const dim3 grid((uint32_t)rows), threads(RopeShape<kDim>::kWaves * kWave);
  if (interleaved) {
    hipLaunchKernelGGL((rope_rows_kernel<kDim, true>), grid, threads, 0, stream, p);
  } else {
    hipLaunchKernelGGL((rope_rows_kernel<kDim, false>), grid, threads, 0, stream, p);
  }
}

}  // namespace
}  // namespace gemma4

using namespace gemma4;

extern "C" {

hipError_t gemma4_rope_frequencies(double *turns, float *amplitude, int32_t rotary_dim,
                                   int32_t exponent_dim, double theta,
                                   Gemma4RopeScaling scaling, double factor,
                                   double original_context, double fast_turns, double slow_turns) {
  if (turns == nullptr || amplitude == nullptr || rotary_dim <= 0 || rotary_dim % 2 != 0 ||
      rotary_dim > 2 * kMaxPairs || exponent_dim < rotary_dim || !(theta > 1.0) ||
      !isfinite(theta) || scaling < GEMMA4_ROPE_PLAIN || scaling > GEMMA4_ROPE_BY_PARTS) {
    return hipErrorInvalidValue;
  }
  const bool scaled = scaling != GEMMA4_ROPE_PLAIN, parts = scaling == GEMMA4_ROPE_BY_PARTS;
  if (scaled && !(factor >= 1.0 && isfinite(factor))) return hipErrorInvalidValue;
  if (scaling == GEMMA4_ROPE_BASE && exponent_dim <= 2) return hipErrorInvalidValue;
  if (parts && !(original_context > 0.0 && isfinite(original_context) && slow_turns >= 0.0 &&
                 fast_turns > slow_turns && isfinite(fast_turns))) {
    return hipErrorInvalidValue;
  }
  constexpr double kTwoPi = 6.283185307179586476925286766559;
  if (scaling == GEMMA4_ROPE_BASE)
    theta *= pow(factor, (double)exponent_dim / (double)(exponent_dim - 2));
  for (int32_t i = 0; i < rotary_dim / 2; ++i) {
    double f = pow(theta, -2.0 * i / exponent_dim) / kTwoPi;
    if (scaling == GEMMA4_ROPE_LINEAR) f /= factor;
    if (parts) {
      const double kept = (original_context * f - slow_turns) / (fast_turns - slow_turns);
      const double part = kept < 0.0 ? 0.0 : (kept > 1.0 ? 1.0 : kept);
      f *= part + (1.0 - part) / factor;
    }
    turns[i] = f;
  }
  *amplitude = parts ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return hipSuccess;
}

hipError_t gemma4_rope_rows_bf16(gemma4_bf16 *d_q_out, gemma4_bf16 *d_k_out, gemma4_bf16 *d_v_out,
                                 const gemma4_bf16 *d_q, const gemma4_bf16 *d_k,
                                 const gemma4_bf16 *d_v, const gemma4_bf16 *d_q_norm_weight,
                                 const gemma4_bf16 *d_k_norm_weight,
                                 const int32_t *d_token_position, const double *d_turns,
                                 float amplitude, int32_t rotary_dim, int32_t interleaved,
                                 int32_t num_heads, int32_t head_dim, int32_t rows,
                                 int64_t q_stride, int64_t kv_stride, hipStream_t stream) {
  if (rows == 0) return hipSuccess;
  const bool geometry = (num_heads == 8 && head_dim == 256) || (num_heads == 1 && head_dim == 512);
  // A launch holds fewer than 2^32 threads.
  if (!geometry || rows < 0 || rows > (1 << 22) || rotary_dim <= 0 || rotary_dim > head_dim ||
      rotary_dim % 16 != 0 || !isfinite(amplitude) || d_q_out == nullptr || d_k_out == nullptr ||
      d_q == nullptr || d_k == nullptr || (d_v != nullptr && d_v_out == nullptr) ||
      d_token_position == nullptr || d_turns == nullptr) {
    return hipErrorInvalidValue;
  }
  const int64_t q_width = (int64_t)kQueryHeads * head_dim, kv_width = (int64_t)num_heads * head_dim;
  if (q_stride == 0) q_stride = q_width;
  if (kv_stride == 0) kv_stride = kv_width;
  const int64_t most = (int64_t)1 << 30;
  if (q_stride < q_width || kv_stride < kv_width || q_stride % kPackElems != 0 ||
      kv_stride % kPackElems != 0 || q_stride > most || kv_stride > most || !aligned(d_q_out, 16) ||
      !aligned(d_k_out, 16) || !aligned(d_v_out, 16) || !aligned(d_q, 16) || !aligned(d_k, 16) ||
      !aligned(d_v, 16) || !aligned(d_q_norm_weight, 16) || !aligned(d_k_norm_weight, 16) ||
      !aligned(d_turns, 8)) {
    return hipErrorInvalidValue;
  }
  RopeParams p{};
  p.q_out = reinterpret_cast<uint16_t *>(d_q_out);
  p.k_out = reinterpret_cast<uint16_t *>(d_k_out);
  p.v_out = reinterpret_cast<uint16_t *>(d_v_out);
  p.q = reinterpret_cast<const uint16_t *>(d_q);
  p.k = reinterpret_cast<const uint16_t *>(d_k);
  p.v = reinterpret_cast<const uint16_t *>(d_v);
  p.q_weight = reinterpret_cast<const uint16_t *>(d_q_norm_weight);
  p.k_weight = reinterpret_cast<const uint16_t *>(d_k_norm_weight);
  p.position = d_token_position;
  p.turns = d_turns;
  p.q_stride = q_stride;
  p.kv_stride = kv_stride;
  p.amplitude = amplitude;
  p.rotary = rotary_dim;
  if (num_heads == 1) {
    launch_rope<512>(p, rows, interleaved != 0, stream);
  } else {
    launch_rope<256>(p, rows, interleaved != 0, stream);
  }
  return hipGetLastError();
}

}  // extern "C"
