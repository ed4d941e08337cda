// The launch of a ragged extension batch in row blocks of a few rows (extend_few.hip).
#pragma once

#include "extend_common.hpp"

namespace gemma4 {

// Blocks of one wave's rows of extend_rows.hip, so that partial sums have that layout.
constexpr ExtendGeometry kFew256 = {16, 16, 64, 32};
constexpr ExtendGeometry kFew512 = {2, 2, 64, 256};
static_assert(kFew256.rows == kExtend256.wave_rows && kFew512.rows == kExtend512.wave_rows);

// LDS accesses of one wave complete in order; this stops the compiler from moving them.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

void launch_extend_few(const ExtendParams &p, hipStream_t stream);

}  // namespace gemma4
