// Division of a position by a run-time divisor that is fixed for a launch
// (page size, pages per sequence): a multiply-high, an add and a shift in place
// of the ~20 instructions of an integer divide.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gemma4 {

// floor(n / d) = (mulhi(n, mul) + n) >> shift with shift = ceil(log2 d) and
// mul = floor(2^32 (2^shift - d) / d) + 1 (Granlund & Montgomery, "Division by
// Invariant Integers using Multiplication", 1994), for n < 2^31: the sum stays
// below 2^32. d >= 1.
struct FastDiv {
  uint32_t d, mul, shift;
};

inline FastDiv make_fast_div(int32_t divisor) {
  FastDiv f;
  f.d = (uint32_t)divisor;
  f.shift = 0;
  while ((1ull << f.shift) < f.d) ++f.shift;
  f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - f.d)) / f.d + 1);
  return f;
}

__host__ __device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &f) {
#if defined(__HIP_DEVICE_COMPILE__)
  return (__umulhi(n, f.mul) + n) >> f.shift;
#else
  return ((uint32_t)(((uint64_t)n * f.mul) >> 32) + n) >> f.shift;
#endif
}
__host__ __device__ __forceinline__ uint32_t fast_mod(uint32_t n, const FastDiv &f) {
  return n - fast_div(n, f) * f.d;
}

}  // namespace gemma4
