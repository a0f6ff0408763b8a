// Activations in 8 bits (qw4_a8): what the kernels that write them (a8_rows.hip) and
// those that read them (a8_linear.hip) share.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "w4a16_common.h"

namespace qw4 {

// The arrays of `a` are there, and it holds rows [row0, row0 + T).
inline int check_a8(const qw4_a8* a, int row0, int T) {
  if (!a || !a->q || !a->scale) return QW4_ERR_NULL;
  if (a->in_f <= 0 || a->in_f % kGroup || a->max_rows < 1) return QW4_ERR_SHAPE;
  if (((uintptr_t)a->q & 15) || ((uintptr_t)a->scale & 3)) return QW4_ERR_ALIGN;
  if (row0 < 0 || T > a->max_rows - row0) return QW4_ERR_SCRATCH;
  return QW4_OK;
}

}  // namespace qw4
