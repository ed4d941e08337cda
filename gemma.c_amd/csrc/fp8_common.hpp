// e4m3 codes of the quantised cache (gfx950 converts the OCP format in
// hardware): a value is code * scale, the scale fixed for a layer's KV head.
#pragma once

#include "gemma4_device.hpp"

namespace gemma4 {

constexpr float kFp8Max = 448.0f;  // the largest e4m3 value
constexpr int kPackCodes = 16;     // codes of a 128-bit pack

// Two values as codes in half a word (the low one, or with kHigh the high one; the
// other half stays as in `old`): the nearest code, ties to the even one, beyond the
// largest value that value; NaN stays NaN. The quotient is the correctly rounded
// one, so a code is what the definition says but for quotients within 2^-24 of a tie.
template <bool kHigh>
__device__ __forceinline__ uint32_t fp8_pair(float a, float b, float scale, uint32_t old) {
  a /= scale;
  b /= scale;
  a = a != a ? a : __builtin_amdgcn_fmed3f(a, -kFp8Max, kFp8Max);
  b = b != b ? b : __builtin_amdgcn_fmed3f(b, -kFp8Max, kFp8Max);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, kHigh);
}
// Four bf16 (two words) as codes.
__device__ __forceinline__ uint32_t fp8_word(uint32_t lo, uint32_t hi, float scale) {
  const uint32_t w = fp8_pair<false>(bf16_lo(lo), bf16_hi(lo), scale, 0);
  return fp8_pair<true>(bf16_lo(hi), bf16_hi(hi), scale, w);
}
// 16 bf16 as codes.
__device__ __forceinline__ uint4 fp8_pack(const uint4 &a, const uint4 &b, float scale) {
  return make_uint4(fp8_word(a.x, a.y, scale), fp8_word(a.z, a.w, scale),
                    fp8_word(b.x, b.y, scale), fp8_word(b.z, b.w, scale));
}

// Two codes (the low half of w, or with kHigh the high one) as a bf16 pair: exact, a
// code has four significant bits.
template <bool kHigh>
__device__ __forceinline__ uint32_t fp8_to_bf16(uint32_t w) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
}

// Scale of a layer's KV head, [num_layers][num_heads]; no array: 1.
__device__ __forceinline__ float fp8_scale(const float *scales, const Gemma4KvCacheConfig &c,
                                           int32_t layer, int32_t head) {
  return scales != nullptr ? scales[layer * c.num_heads + head] : 1.0f;
}

}  // namespace gemma4
