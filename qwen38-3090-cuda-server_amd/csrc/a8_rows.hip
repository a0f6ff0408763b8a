// Rows of activations in 8 bits: qw4_a8_quantize, qw4_a8_rmsnorm and their inverse.
//
// A group of 128 inputs is 16 lanes of 8. A = max |v| over the group (a maximum of the
// bits, in which NaN is the largest), scale = A / 127, q = RNE(v 127 / A): the product
// and the rounding are one fma against 1.5 2^23, whose lowest byte is then q. 127 / A is
// rounded up: v = A / 2, which bf16 rows meet constantly, is 63.5 or as little above it as
// fp32 tells, and becomes 64, the even one. Of bf16 values no other quotient is so close to
// the middle of two codes that the rounding of 127 / A moves it across (all pairs of
// mantissas are tested); of a norm's fp32 values one within 2^-23 of itself may go either way.
// The codes of a word's 8 inputs are the bytes {0, 4, 1, 5} and {2, 6, 3, 7}, as the low
// and the high nibbles of a packed weight word hold them: a product reads its operand
// 16 bytes at a time with no shuffle.
//
// All are bound by HBM from some 4 MB on, by the launch below: 4096 x 5120 with residual 28 us
// (147 MB, 5.2 TB/s; a large copy reaches 4.7), quantized alone 15, back to bf16 12; one row
// 2.4 / 1.7 / 1.5 us on the GPU.
#include <hip/hip_runtime.h>

#include <cstring>

#include "../../include/qwen_w4a16.h"
#include "a8.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}

// Largest of the 16 lanes of a DPP row.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, dpp<0xB1>(v));    // quad_perm [1, 0, 3, 2]
  v = max(v, dpp<0x4E>(v));    // quad_perm [2, 3, 0, 1]
  v = max(v, dpp<0x141>(v));   // row_half_mirror
  return max(v, dpp<0x140>(v));   // row_mirror
}

// Below this a group counts as zeros: 127 / A stays finite, and no output of a product
// over such values is anywhere near bf16's or fp32's range.
constexpr float kA8Least = 0x1p-100f;

// The codes of a lane's 8 values and the scale of its group, whose 16 lanes (a DPP row)
// all call this. The lane's 8 bytes of the row go to its words: bytes 8 l .. 8 l + 7 of a
// 32-byte chunk are words of lanes 2 l, 2 l + 1 of four (first halves: l = 0, 1; second
// halves: l = 2, 3).
__device__ __forceinline__ u32x2 a8_codes(const float (&v)[8], int lane, float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = row16_max(top);
  const float a = __uint_as_float(top);
  const bool some = a >= kA8Least && top < 0x7f800000u;
  scale = some ? a / 127.f : top >= 0x7f800000u ? __builtin_nanf("") : 0.f;
  float r = some ? 127.f / a : 0.f;
  if (__builtin_fmaf(-r, a, 127.f) > 0.f && some) r = __uint_as_float(__float_as_uint(r) + 1);   // the fma is exact
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(__builtin_fmaf(v[e], r, 12582912.f));
  // byte 0 of four registers into one: perm's selector 0..3 takes the second operand's bytes
  auto four = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
    const uint32_t lo = __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b3, b2, 0x0c0c0400u);
    return lo | (hi << 16);
  };
  const uint32_t even = four(b[0], b[4], b[1], b[5]), odd = four(b[2], b[6], b[3], b[7]);
  const bool first = (lane & 3) < 2;
  const uint32_t e0 = dpp<0x88>(even), o0 = dpp<0x88>(odd);   // quad_perm [0, 2, 0, 2]
  const uint32_t e1 = dpp<0xDD>(even), o1 = dpp<0xDD>(odd);   // quad_perm [1, 3, 1, 3]
  return {first ? e0 : o0, first ? e1 : o1};
}

__device__ __forceinline__ void unpack8(float (&v)[8], const u32x4& x) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    v[2 * c] = bf16_bits_to_f32(x[c] & 0xffffu);
    v[2 * c + 1] = bf16_bits_to_f32(x[c] >> 16);
  }
}

constexpr int kA8Threads = 256;
constexpr int kA8Units = kA8Threads / 16;   // groups of a workgroup

// 16 lanes a (row, group).
__global__ __launch_bounds__(kA8Threads) void k_a8_quantize(int8_t* q, float* scale, const uint16_t* x,
                                                            size_t ld, uint32_t units, uint32_t G,
                                                            int max_rows) {
  const uint32_t u = blockIdx.x * kA8Units + (threadIdx.x >> 4);
  if (u >= units) return;
  const uint32_t row = u / G, g = u - row * G;
  const int l = threadIdx.x & 15;
  float v[8], s;
  unpack8(v, *reinterpret_cast<const u32x4*>(x + row * ld + g * kGroup + 8 * l));
  const u32x2 codes = a8_codes(v, l, s);
  *reinterpret_cast<u32x2*>(q + ((size_t)row * G + g) * kGroup + 8 * l) = codes;
  if (l == 0) scale[(size_t)g * max_rows + row] = s;
}

// qw4_rmsnorm's sum of squares and inverse (norm_sumsq, norm_inv), then the codes. One
// workgroup of T threads per row; thread t stands for the virtual threads t + T k.
// Chunks behind the first 1024 (rows beyond 8192) are read again by the thread that
// read them first -- with a residual, as it wrote them.
template <int T, int PER, bool RES>
__global__ __launch_bounds__(T) void k_a8_rmsnorm(int8_t* q, float* scale, uint16_t* h_out, const uint16_t* h,
                                                  const uint16_t* res, const uint16_t* w, int dim,
                                                  int max_rows, float eps) {
  const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int kc = dim / 8;
  const u32x4* hr = reinterpret_cast<const u32x4*>(h + (size_t)row * dim);
  const u32x4* rr = reinterpret_cast<const u32x4*>(res + (size_t)row * dim);
  const u32x4* wr = reinterpret_cast<const u32x4*>(w);
  u32x4* orow = reinterpret_cast<u32x4*>(h_out + (size_t)row * dim);
  __shared__ float vsum[kNormVWaves];
  auto add = [](u32x4 a, const u32x4& b) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      a[e] = pack_bf16x2(bf16_bits_to_f32(a[e] & 0xffffu) + bf16_bits_to_f32(b[e] & 0xffffu),
                         bf16_bits_to_f32(a[e] >> 16) + bf16_bits_to_f32(b[e] >> 16));
    return a;
  };
  u32x4 hv[PER], rv[PER], wv[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = min(t + T * k, kc - 1);
    hv[k] = hr[i];
    if (RES) rv[k] = rr[i];
    wv[k] = wr[i];
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    float ss = 0.f;
    if (t + T * k < kc) {
      if (RES) orow[t + T * k] = hv[k] = add(hv[k], rv[k]);
      ss = norm_sumsq(0.f, hv[k]);
    }
    for (int i = t + T * k + kNormVThreads; i < kc; i += kNormVThreads) {
      u32x4 v = hr[i];
      if (RES) orow[i] = v = add(v, rr[i]);
      ss = norm_sumsq(ss, v);
    }
    ss = norm_wave_sum(ss);
    if (lane == 0) vsum[wave + (T / 64) * k] = ss;
  }
  if (t < kNormVWaves - PER * (T / 64)) vsum[PER * (T / 64) + t] = 0.f;   // virtual waves past the row
  __syncthreads();
  const float inv = norm_inv(vsum, dim, eps);
  auto store = [&](int i, const u32x4& v, const u32x4& g) {
    float y[8], s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[2 * e] = rmsnorm_f32(v[e], g[e], inv);
      y[2 * e + 1] = rmsnorm_f32(v[e] >> 16, g[e] >> 16, inv);
    }
    const u32x2 codes = a8_codes(y, i, s);
    *reinterpret_cast<u32x2*>(q + (size_t)row * dim + 8 * i) = codes;
    if ((i & 15) == 0) scale[(size_t)(i >> 4) * max_rows + row] = s;
  };
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (t + T * k < kc) store(t + T * k, hv[k], wv[k]);
  const u32x4* again = RES ? orow : hr;
  for (int i = t + kNormVThreads; i < kc; i += T) store(i, again[i], wr[i]);
}

// 8 outputs a thread: the two words that hold them.
__global__ __launch_bounds__(kA8Threads) void k_a8_dequant(uint16_t* dst, const int8_t* q, const float* scale,
                                                           uint32_t chunks, uint32_t kc, int max_rows) {
  const uint32_t c = blockIdx.x * kA8Threads + threadIdx.x;
  if (c >= chunks) return;
  const uint32_t row = c / kc, i = c - row * kc;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(q + (size_t)row * kc * 8 + (i >> 2) * 32);
  const uint32_t even = words[i & 3], odd = words[4 + (i & 3)];
  const float s = scale[(size_t)(i >> 4) * max_rows + row];
  auto f = [&](uint32_t w, int b) { return (float)(int8_t)(w >> (8 * b)) * s; };
  reinterpret_cast<u32x4*>(dst)[c] = u32x4{pack_bf16x2(f(even, 0), f(even, 2)), pack_bf16x2(f(odd, 0), f(odd, 2)),
                                           pack_bf16x2(f(even, 1), f(even, 3)), pack_bf16x2(f(odd, 1), f(odd, 3))};
}

// Rows of one launch whose units of work (a row's `per`) stay below 2^27.
int launch_rows(size_t per) { return (int)std::max<size_t>(1, (1u << 27) / per); }

template <bool RES>
void launch_norm(const qw4_a8& a, uint16_t* o, const uint16_t* h, const uint16_t* r, const uint16_t* w, int T,
                 float eps, hipStream_t s) {
  const int dim = a.in_f;
  // 1024 threads a row while rows are few: 512 x 5120 with residual 5.9 us, with 256 threads 6.8;
  // 600 7.5 and 7.9, but without residual 5.6 and 5.5, 2047 x 4096 11.9 and 9.3
  if (T <= 512) {
    k_a8_rmsnorm<kNormVThreads, 1, RES><<<T, kNormVThreads, 0, s>>>(a.q, a.scale, o, h, r, w, dim, a.max_rows, eps);
    return;
  }
  launch_rows_of(T, 1 << 23, [&](int first, int n) {
    const size_t at = (size_t)first * dim;
    auto go = [&](auto kernel) {
      kernel<<<n, kA8Threads, 0, s>>>(a.q + at, a.scale + first, RES ? o + at : nullptr, h + at,
                                      RES ? r + at : nullptr, w, dim, a.max_rows, eps);
    };
    if (dim <= 8 * kA8Threads)
      go(k_a8_rmsnorm<kA8Threads, 1, RES>);
    else if (dim <= 16 * kA8Threads)
      go(k_a8_rmsnorm<kA8Threads, 2, RES>);
    else
      go(k_a8_rmsnorm<kA8Threads, 4, RES>);
  });
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_a8_alloc(qw4_a8* a, int max_rows, int in_f) {
  if (!a) return QW4_ERR_NULL;
  std::memset(a, 0, sizeof(*a));
  if (max_rows < 1 || in_f <= 0 || in_f % kGroup) return QW4_ERR_SHAPE;
  qw4_a8 b{};
  hipError_t e = hipMalloc(&b.q, (size_t)max_rows * in_f);
  if (e == hipSuccess) e = hipMalloc(&b.scale, (size_t)max_rows * (in_f / kGroup) * 4);
  if (e != hipSuccess) {
    set_hip_error((int)e);
    (void)hipGetLastError();
    if (b.q) (void)hipFree(b.q);
    return QW4_ERR_NOMEM;
  }
  b.max_rows = max_rows;
  b.in_f = in_f;
  *a = b;
  return QW4_OK;
}

int qw4_a8_free(qw4_a8* a) {
  if (!a) return QW4_ERR_NULL;
  if (a->q) (void)hipFree(a->q);
  if (a->scale) (void)hipFree(a->scale);
  std::memset(a, 0, sizeof(*a));
  return QW4_OK;
}

int qw4_a8_quantize(const qw4_a8* a, const uint16_t* x, int ld, int T, void* stream) {
  if (T < 0) return QW4_ERR_M;
  const int st = check_a8(a, 0, T);
  if (st) return st;
  if (ld < a->in_f || ld % 8) return QW4_ERR_SHAPE;
  if (T == 0) return QW4_OK;
  if (!x) return QW4_ERR_NULL;
  if ((uintptr_t)x & 15) return QW4_ERR_ALIGN;
  const uint32_t G = (uint32_t)a->in_f / kGroup;
  launch_rows_of(T, launch_rows(G), [&](int first, int n) {
    const uint32_t units = (uint32_t)n * G;
    k_a8_quantize<<<(units + kA8Units - 1) / kA8Units, kA8Threads, 0, (hipStream_t)stream>>>(
        a->q + (size_t)first * a->in_f, a->scale + first, x + (size_t)first * ld, (size_t)ld, units, G, a->max_rows);
  });
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

int qw4_a8_rmsnorm(const qw4_a8* a, uint16_t* h_out, const uint16_t* h, const uint16_t* residual,
                   const uint16_t* w, int T, float eps, void* stream) {
  if (T < 0) return QW4_ERR_M;
  const int st = check_a8(a, 0, T);
  if (st) return st;
  if (T == 0) return QW4_OK;
  if (!h || !w || (residual && !h_out)) return QW4_ERR_NULL;
  if (((uintptr_t)h_out | (uintptr_t)h | (uintptr_t)residual | (uintptr_t)w) & 15) return QW4_ERR_ALIGN;
  if (residual)
    launch_norm<true>(*a, h_out, h, residual, w, T, eps, (hipStream_t)stream);
  else
    launch_norm<false>(*a, nullptr, h, nullptr, w, T, eps, (hipStream_t)stream);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

int qw4_a8_dequant_rows(uint16_t* dst, const qw4_a8* a, int row0, int nrows, void* stream) {
  if (nrows < 0) return QW4_ERR_SHAPE;
  const int st = check_a8(a, row0, nrows);
  if (st) return st == QW4_ERR_SCRATCH ? QW4_ERR_SHAPE : st;
  if (nrows == 0) return QW4_OK;
  if (!dst) return QW4_ERR_NULL;
  if ((uintptr_t)dst & 15) return QW4_ERR_ALIGN;
  const uint32_t kc = (uint32_t)a->in_f / 8;
  launch_rows_of(nrows, launch_rows(kc), [&](int first, int n) {
    const uint32_t chunks = (uint32_t)n * kc;
    const size_t at = (size_t)row0 + first;
    k_a8_dequant<<<(chunks + kA8Threads - 1) / kA8Threads, kA8Threads, 0, (hipStream_t)stream>>>(
        dst + (size_t)first * a->in_f, a->q + at * a->in_f, a->scale + at, chunks, kc, a->max_rows);
  });
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // extern "C"
