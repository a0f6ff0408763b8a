// Operands of the fp16 tile (G2F16, gemm_tile.h): activation rows times a power of two,
// and the exponents that take it back. One launch (2^22 rows each): a workgroup a row of x, then
// workgroups of 256 weight rows, whose largest scale over their groups sets the
// exponent. Bound by x read and written once (the second reading of a row is cached)
// and the scales, 1/26 of the weights.
#include <hip/hip_runtime.h>

#include "gemm_tile.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {   // of two 16-bit halves each
  return max(a & 0xffffu, b & 0xffffu) | max(a & 0xffff0000u, b & 0xffff0000u);
}

__global__ __launch_bounds__(kThreads) void k_half_rows(uint16_t* out, int* rexp, int* cexp,
                                                        const uint16_t* x, int T, int K,
                                                        const uint16_t* sc, int N, int G) {
  const int t = threadIdx.x;
  if ((int)blockIdx.x >= T) {
    const int n = ((int)blockIdx.x - T) * kThreads + t;
    if (n >= N) return;
    const uint16_t* s = sc + (size_t)(n / kTileN) * G * kMetaU16 + n % kTileN;
    uint32_t m = 0;
#pragma unroll 8
    for (int g = 0; g < G; ++g) m = max(m, s[(size_t)g * kMetaU16] & 0x7fffu);
    // the row's largest scale in [2^10, 2^11): its weights stay below 2^15
    cexp[n] = max((int)(m >> 7) - 127 - 10, -126);
    return;
  }
  __shared__ uint32_t part[kThreads / 64];
  const u32x4* row = reinterpret_cast<const u32x4*>(x + (size_t)blockIdx.x * K);
  const int chunks = K / 8;
  uint32_t m = 0;
  for (int i = t; i < chunks; i += kThreads) {
    const u32x4 v = row[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max_pair(m, v[e] & 0x7fff7fffu);
  }
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if ((t & 63) == 0) part[t >> 6] = m;
  __syncthreads();
  m = max(max(part[0], part[1]), max(part[2], part[3]));
  // largest value in [2^14, 2^15); Inf and NaN stay what they are
  const int e = max((int)(m >> 7) - 127 - 14, -126);
  const float by = __builtin_ldexpf(1.f, -e);
  if (t == 0) rexp[blockIdx.x] = e;
  u32x4* to = reinterpret_cast<u32x4*>(out + (size_t)blockIdx.x * K);
  for (int i = t; i < chunks; i += kThreads) {
    const u32x4 v = row[i];
    u32x4 o;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const G2F16::f16x2 h = {(_Float16)(bf16_bits_to_f32(v[c] & 0xffffu) * by),
                              (_Float16)(bf16_bits_to_f32(v[c] >> 16) * by)};
      o[c] = __builtin_bit_cast(uint32_t, h);
    }
    to[i] = o;
  }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t half_rows_bytes(int T, const qw4_weights* w) {
  return align256((size_t)T * w->in_f * 2) + align256((size_t)T * 4) + align256((size_t)w->out_f * 4);
}

HalfRows half_rows(void* buf, const uint16_t* x, int T, const qw4_weights* w, hipStream_t s) {
  char* p = static_cast<char*>(buf);
  uint16_t* out = reinterpret_cast<uint16_t*>(p);
  int* rexp = reinterpret_cast<int*>(p + align256((size_t)T * w->in_f * 2));
  int* cexp = reinterpret_cast<int*>(reinterpret_cast<char*>(rexp) + align256((size_t)T * 4));
  launch_rows_of(T, 1 << 22, [&](int first, int n) {
    const size_t at = (size_t)first * w->in_f;
    const int N = first ? 0 : w->out_f;   // the weight rows once
    k_half_rows<<<n + (N + kThreads - 1) / kThreads, kThreads, 0, s>>>(
        out + at, rexp + first, cexp, x + at, n, w->in_f, w->scale, N, w->num_groups);
  });
  return {out, rexp, cexp};
}

}  // namespace qw4

extern "C" size_t qw4_epilogue_workspace(const qw4_weights* w, int rows) {
  if (!w || w->in_f <= 0 || w->out_f <= 0 || rows < 0) return 0;
  return qw4::half_rows_bytes(rows, w);
}
