// Activations in 8 bits (qw4_a8): what the kernels that write them (a8_rows.hip) and
// those that read them (a8_linear.hip) share.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "epilogue.h"
#include "w4a16_common.h"

namespace qw4 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// Outputs of a product: bf16 with an epilogue, gate and up joined, fp32.
enum { A8_EPI = 0, A8_GLU = 1, A8_F32 = 2 };

struct A8Args {
  const uint32_t* qw;
  const uint16_t* sc;    // (scale, zero-point) records
  const int8_t* q;
  const float* scale;
  void* y;               // bf16, or fp32 (A8_F32)
  int M, N, K, G, max_rows, ld;
  Epilogue epi;
};

// Four weights q - z of each byte's low nibble: 128 + q - z borrows from no other byte.
__device__ __forceinline__ uint32_t a8_less(uint32_t nib, uint32_t z) {
  return ((nib | 0x80808080u) - z) ^ 0x80808080u;
}

// A group's integer sum starts as the bits of M = 1.5 2^23, so that, read as a float, it is M +
// sum: t = fma(f, sw, -M sw) is the sum scaled by the weight's scale, rounded once, for M sw is
// exact for the 8 bits of a bf16 sw (below 2^104, from where it is Inf). The row's scale, of 24
// bits, comes second.
constexpr float kA8Magic = 12582912.f;
constexpr int kA8Start = 0x4B400000;

// The kernel for few rows (a8_few.h): launches it and returns true, or returns false
// where it does not apply.
bool a8_few(int out, const A8Args& a, int cus, hipStream_t st);
bool a8_few_epi(const A8Args& a, int P, int U, bool small, hipStream_t st);
bool a8_few_f32(const A8Args& a, int P, int U, bool small, hipStream_t st);

// The arrays of `a` are there, and it holds rows [row0, row0 + T).
inline int check_a8(const qw4_a8* a, int row0, int T) {
  if (!a || !a->q || !a->scale) return QW4_ERR_NULL;
  if (a->in_f <= 0 || a->in_f % kGroup || a->max_rows < 1) return QW4_ERR_SHAPE;
  if (((uintptr_t)a->q & 15) || ((uintptr_t)a->scale & 3)) return QW4_ERR_ALIGN;
  if (row0 < 0 || T > a->max_rows - row0) return QW4_ERR_SCRATCH;
  return QW4_OK;
}

}  // namespace qw4
