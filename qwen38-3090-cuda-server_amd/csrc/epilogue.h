// The epilogue of a product: v = acc + bias, f(v), + residual, one rounding to bf16.
// Everything before the rounding is fp32.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "w4a16_common.h"

namespace qw4 {

struct Epilogue {
  const uint16_t* bias;   // per weight row, or null
  const uint16_t* res;    // rows of the output's width, or null (may be the output)
  int act;                // QW4_ACT_*
  int up;                 // QW4_ACT_SWIGLU: weight rows from a gate row to its up row
};

// exp and 1 / x at the hardware's rate, a third of the code of the exact ones, of which an
// epilogue holds dozens. exp's argument in powers of two is rounded, so exp is off by
// |v| 2^-24 (2^-18 at |v| = 80) on top of the instruction's 2^-22: far below the output's
// rounding, 2^-8.
__device__ __forceinline__ float fast_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.4426950408889634f); }
__device__ __forceinline__ float act_silu(float v) {
  return v * __builtin_amdgcn_rcpf(1.f + fast_exp(-v));
}

// v erfc(-v / sqrt 2) / 2: with 1 + erf the terms would cancel for negative v. erfc(z) =
// t exp(-z^2 + P(t)), t = 1 / (1 + z / 2), z >= 0, by the Chebyshev fit of Press et al.,
// Numerical Recipes, section 6.2 (the fit's relative error is below 1.2e-7; exp adds
// its argument's rounding, z^2 2^-24).
__device__ __forceinline__ float act_gelu(float v) {
  const float z = fabsf(v) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f, z, 1.f));
  float p = 0.17087277f;
  p = __builtin_fmaf(p, t, -0.82215223f);
  p = __builtin_fmaf(p, t, 1.48851587f);
  p = __builtin_fmaf(p, t, -1.13520398f);
  p = __builtin_fmaf(p, t, 0.27886807f);
  p = __builtin_fmaf(p, t, -0.18628806f);
  p = __builtin_fmaf(p, t, 0.09678418f);
  p = __builtin_fmaf(p, t, 0.37409196f);
  p = __builtin_fmaf(p, t, 1.00002368f);
  p = __builtin_fmaf(p, t, -1.26551223f);
  const float half = 0.5f * t * fast_exp(__builtin_fmaf(-z, z, p));   // erfc(z) / 2
  return v * (v < 0.f ? half : 1.f - half);
}

// v / (1 + exp(-2 u)) = v (1 + tanh u) / 2, without its cancellation
__device__ __forceinline__ float act_gelu_tanh(float v) {
  const float u2 = 1.5957691216057308f * __builtin_fmaf(0.044715f * v * v, v, v);
  return v * __builtin_amdgcn_rcpf(1.f + fast_exp(-u2));
}

// v[0] = f(v[0]), gated: silu(v[0]) v[1]; the act is the same for a whole launch.
template <bool GLU, int N>
__device__ __forceinline__ void epilogue_act(float (&v)[GLU ? 2 : 1][N], int act) {
  if constexpr (GLU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = act_silu(v[0][i]) * v[1][i];
  } else if (act == QW4_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = act_silu(v[0][i]);
  } else if (act == QW4_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = act_gelu(v[0][i]);
  } else if (act == QW4_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = act_gelu_tanh(v[0][i]);
  }
}

// Bias of 8 columns from `col` of a wave (16-byte aligned), zeros without one.
template <bool GLU>
__device__ __forceinline__ void load_bias(float (&b)[GLU ? 2 : 1][8], const Epilogue& e, int col) {
#pragma unroll
  for (int j = 0; j < (GLU ? 2 : 1); ++j) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (e.bias) v = *reinterpret_cast<const u32x4*>(e.bias + j * e.up + col);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      b[j][2 * c] = bf16_bits_to_f32(v[c] & 0xffffu);
      b[j][2 * c + 1] = bf16_bits_to_f32(v[c] >> 16);
    }
  }
}

// bf16(v + residual) of 8 columns.
__device__ __forceinline__ u32x4 add_round8(const float (&v)[8], const u32x4& res) {
  u32x4 o;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    o[c] = pack_bf16x2(v[2 * c] + bf16_bits_to_f32(res[c] & 0xffffu),
                       v[2 * c + 1] + bf16_bits_to_f32(res[c] >> 16));
  return o;
}

// The prefill GEMM with an epilogue (gemm.hip), over checked arguments.
int gemm_epilogue(uint16_t* y, const qw4_weights* w, const uint16_t* x, int M, qw4_workspace* ws,
                  const Epilogue& e, void* stream);

// Rows up to which a product with a weight of out_f rows uses it exactly or, with a
// workspace, to 11 bits at least (linear.hip; qw4_linear_max_t without its override).
int exact_rows(int out_f, int in_f);

}  // namespace qw4
