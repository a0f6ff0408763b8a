// Products of activations in 8 bits and INT4 weights (qw4_a8_linear).
//
//   y[m][n] = act(sum_g sx[m][g] sw[n][g] (sum_{k in g} (qw[n][k] - z[n][g]) qx[m][k]) + bias[n]) + res[m][n]
//
// The inner sum is exact in int32 (at most 128 15 127 = 243840) on v_mfma_i32_32x32x32_i8:
// the low nibbles of a packed word less their zero point are four int8 weights, the high
// ones four more, and the activation rows hold their codes in that order. A group's sums
// are scaled into fp32 accumulators.
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "a8.h"
#include "epilogue.h"
#include "w4a16_common.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct A8Args {
  const uint32_t* qw;
  const uint16_t* sc;
  const uint16_t* zr;
  const int8_t* q;
  const float* scale;
  void* y;               // bf16, or fp32 (F32)
  int M, N, K, G, max_rows, ld;
  Epilogue epi;
};

// Four weights q - z of each byte's low nibble: 128 + q - z borrows from no other byte.
__device__ __forceinline__ uint32_t a8_less(uint32_t nib, uint32_t z) {
  return ((nib | 0x80808080u) - z) ^ 0x80808080u;
}

// A wave computes 32 columns (rows of W) x 32 rows of x; gated, the up columns too.
// MFMA layout (A: weights): lane l holds row l % 32, inputs 16 (l / 32).. of an operand;
// of the result column l % 32 (a row of x), rows 8 j + 4 (l / 32) + i.
template <bool GLU, bool F32>
__global__ __launch_bounds__(64) void k_a8_simple(A8Args a) {
  const int lane = threadIdx.x, r = lane & 31, h = lane >> 5;
  const int n0 = blockIdx.x * 32, m = blockIdx.y * 32 + r;
  const int row = min(m, a.M - 1);
  constexpr int NP = GLU ? 2 : 1;
  float acc[NP][16] = {};
  for (int g = 0; g < a.G; ++g) {
    const u32x4* xr = reinterpret_cast<const u32x4*>(a.q + (size_t)row * a.K + g * kGroup);
    const float sx = a.scale[(size_t)g * a.max_rows + row];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int n = n0 + p * a.epi.up, tile = n / kTileN, b = (n % kTileN) / 32;
      const size_t blk = (size_t)tile * a.G + g;
      const int pos = tile_pos_of_row(32 * b + r);
      const uint32_t z = (a.zr[blk * 16 + (32 * b + r) / 4] >> (4 * (r & 3))) & 15u;
      i32x16 c = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 w = reinterpret_cast<const u32x4*>(a.qw + blk * kWordsPerBlock)[(2 * s + h) * 64 + pos];
        u32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = a8_less(w[i] & 0x0F0F0F0Fu, z * 0x01010101u);
          hi[i] = a8_less((w[i] >> 4) & 0x0F0F0F0Fu, z * 0x01010101u);
        }
        c = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, lo),
                                                  __builtin_bit_cast(i32x4, xr[2 * (2 * s + h)]), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, hi),
                                                  __builtin_bit_cast(i32x4, xr[2 * (2 * s + h) + 1]), c, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sw = bf16_bits_to_f32(a.sc[blk * kMetaU16 + 32 * b + 8 * j + 4 * h + i]);
          acc[p][4 * j + i] = __builtin_fmaf((float)c[4 * j + i] * sx, sw, acc[p][4 * j + i]);
        }
    }
  }
  if (m >= a.M) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = n0 + 8 * j + 4 * h;
    const size_t at = (size_t)m * a.ld + col;
    if constexpr (F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) =
          f32x4{acc[0][4 * j], acc[0][4 * j + 1], acc[0][4 * j + 2], acc[0][4 * j + 3]};
    } else {
      float v[NP][4];
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[p][i] = acc[p][4 * j + i] + (a.epi.bias ? bf16_bits_to_f32(a.epi.bias[p * a.epi.up + col + i]) : 0.f);
      epilogue_act<GLU>(v, a.epi.act);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[0][i] += a.epi.res ? bf16_bits_to_f32(a.epi.res[at + i]) : 0.f;
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + at) =
          u32x2{pack_bf16x2(v[0][0], v[0][1]), pack_bf16x2(v[0][2], v[0][3])};
    }
  }
}

int check_call(const void* y, const qw4_weights* w, const qw4_a8* a, int T) {
  int st = check_weights_public(w);
  if (st) return st;
  if (!y) return QW4_ERR_NULL;
  if (T < 1) return QW4_ERR_M;
  st = check_a8(a, 0, T);
  if (st) return st;
  if (a->in_f != w->in_f) return QW4_ERR_SHAPE;
  if ((uintptr_t)y & 15) return QW4_ERR_ALIGN;
  return QW4_OK;
}

A8Args args_of(void* y, const qw4_weights* w, const qw4_a8* a, int T, const Epilogue& e) {
  return {w->qweight, w->scale, w->zeros, a->q, a->scale, y, T, w->out_f, w->in_f, w->num_groups,
          a->max_rows, w->out_f - e.up, e};
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_a8_linear(uint16_t* y, const qw4_weights* w, const qw4_a8* a, int T, const uint16_t* bias, int act,
                  const uint16_t* residual, qw4_workspace* ws, void* stream) {
  const int st = check_call(y, w, a, T);
  if (st) return st;
  if (act < QW4_ACT_NONE || act > QW4_ACT_SWIGLU) return QW4_ERR_ACT;
  const bool glu = act == QW4_ACT_SWIGLU;
  if (glu && w->out_f % (2 * kTileN)) return QW4_ERR_SHAPE;
  if (((uintptr_t)bias | (uintptr_t)residual) & 15) return QW4_ERR_ALIGN;
  (void)ws;
  const A8Args g = args_of(y, w, a, T, Epilogue{bias, residual, act, glu ? w->out_f / 2 : 0});
  const dim3 grid(g.ld / 32, (T + 31) / 32);
  if (glu)
    k_a8_simple<true, false><<<grid, 64, 0, (hipStream_t)stream>>>(g);
  else
    k_a8_simple<false, false><<<grid, 64, 0, (hipStream_t)stream>>>(g);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

int qw4_a8_linear_f32(float* y, const qw4_weights* w, const qw4_a8* a, int T, qw4_workspace* ws, void* stream) {
  const int st = check_call(y, w, a, T);
  if (st) return st;
  (void)ws;
  const A8Args g = args_of(y, w, a, T, Epilogue{});
  k_a8_simple<false, true><<<dim3(g.ld / 32, (T + 31) / 32), 64, 0, (hipStream_t)stream>>>(g);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // extern "C"
