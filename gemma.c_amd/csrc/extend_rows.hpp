// The launch of a ragged extension batch's rows (extend_rows.hip).
#pragma once

#include "extend_common.hpp"

namespace gemma4 {

void launch_extend_rows(const ExtendParams &p, hipStream_t stream);

}  // namespace gemma4
