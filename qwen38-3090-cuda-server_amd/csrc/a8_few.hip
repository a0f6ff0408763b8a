// Products of few rows in 8 bits (1 to 16, for shorter K to 64, in one reading of the
// weights): qw4_a8_linear's decode, verify and small batches. HBM-bound.
//
// Workgroup p owns whole units (S row quads of a tile, 16 or 32 weight rows, over all of
// K); wave w takes the groups w, w + 8, ... and the units are summed over the waves in
// wave order, as in the bf16 kernel for few rows. A wave meets the same groups in every
// unit, so it holds their codes: 8 registers a group and 16 rows, half of bf16's, and in
// the order that the nibbles of a weight word have, so that they are MFMA operands as
// they lie in memory and the weights stream past them through LDS-DMA slots, D items
// (a group of a unit) ahead, across units. The scales of all rows and groups lie in LDS.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/qwen_w4a16.h"
#include "a8.h"
#include "skinny.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

constexpr int kFewW = 8;   // waves

template <int MB, int S>
constexpr int few_buffers() { return MB * S <= 4 ? 2 : 1; }   // of the waves' sums

// Row m, columns n0 + i of a unit (g: its gate sums).
template <int OUT, int S>
__device__ __forceinline__ void few_emit(const A8Args& a, int m, int n0, const float (&v)[S], const float (&g)[S]) {
  if (m >= a.M) return;
  const size_t at = (size_t)m * a.ld + n0;
  if constexpr (OUT == A8_F32) {
    float* y = static_cast<float*>(a.y) + at;
#pragma unroll
    for (int i = 0; i < S; ++i) y[i] = v[i];
  } else {
    constexpr bool kGlu = OUT == A8_GLU;
    float f[kGlu ? 2 : 1][S], b[kGlu ? 2 : 1][S], r[S];
#pragma unroll
    for (int j = 0; j < (kGlu ? 2 : 1); ++j) {
      load_cols<S>(b[j], a.epi.bias, (size_t)n0 + j * a.epi.up);
#pragma unroll
      for (int i = 0; i < S; ++i) f[j][i] = (kGlu && j == 0 ? g[i] : v[i]) + b[j][i];
    }
    load_cols<S>(r, a.epi.res, at);
    epilogue_act<kGlu, S>(f, a.epi.act);
    uint16_t* y = static_cast<uint16_t*>(a.y) + at;
    if constexpr (S == 1) {
      y[0] = to_bf16(f[0][0] + r[0]);
    } else {
#pragma unroll
      for (int i = 0; i < S / 2; ++i)
        reinterpret_cast<uint32_t*>(y)[i] = pack_bf16x2(f[0][2 * i] + r[2 * i], f[0][2 * i + 1] + r[2 * i + 1]);
    }
  }
}

struct FewArgs {
  A8Args a;
  int P, U;
};

template <int OUT, int S, int NG, int D, int MB>
__global__ __launch_bounds__(64 * kFewW, 2) void k_a8_few(FewArgs f) {
  using L = DmaSlot<4, S>;
  constexpr int W = kFewW, kL = L::kLoads, kBuf = few_buffers<MB, S>();
  constexpr uint32_t kPer = 4 / S;
  constexpr bool kGlu = OUT == A8_GLU;
  const A8Args& a = f.a;
  __shared__ f32x4 red[W][kBuf * MB * S * 64];
  extern __shared__ u32x4 few_lds[];   // the waves' slots, then the scales [G][16 MB]
  float* const sxl = reinterpret_cast<float*>(few_lds + W * D * L::kUnits);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4, zsh = 16 * (c & 1);
  SkinnyRsrc rs;
  rs.qw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(a.qw), 0, (int)((uint32_t)(a.N / kTileN) * a.G * 4096u),
                                            0x00020000);
  rs.sc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.sc), 0,
                                            (int)((uint32_t)(a.N / kTileN) * a.G * (uint32_t)kMetaBytes), 0x00020000);
  rs.x = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.q), 0, (int)((uint32_t)a.M * (uint32_t)a.K), 0x00020000);
  const uint32_t wbase = Fmt<4>::woff(q, c);
  // gated: units 2v (gate v) and 2v + 1 (its up unit), never split
  const int half = kGlu ? f.U / 2 : f.U, p = blockIdx.x;
  const int u0 = (kGlu ? 2 : 1) * (int)((long long)p * half / f.P), u1 = (kGlu ? 2 : 1) * (int)((long long)(p + 1) * half / f.P);
  auto real_unit = [&](int v) { return kGlu ? (v >> 1) + (v & 1) * half : v; };
  const int nw = wave < a.G ? (a.G - 1 - wave) / W + 1 : 0;   // groups of this wave (<= NG)
  const int T = nw * (u1 - u0);                                // its items

  // Codes of this wave's groups: row 16 mb + c, chunk q, its two halves (rows past M are
  // zeros without traffic).
  u32x4 x[NG][MB][2];
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[i][mb][h] = u32x4{0u, 0u, 0u, 0u};
        if (i < nw && 16 * mb < a.M)
          x[i][mb][h] = __builtin_amdgcn_raw_buffer_load_b128(
              rs.x, (uint32_t)(16 * mb + c) * (uint32_t)a.K + (uint32_t)(32 * q + 16 * h), (uint32_t)(wave + W * i) * 128u, 0);
      }
  for (int i = threadIdx.x; i < a.G * 16 * MB; i += 64 * W) {
    const int g = i / (16 * MB), m = i - g * (16 * MB);
    sxl[i] = m < a.M ? a.scale[(size_t)g * a.max_rows + m] : 0.f;
  }
  __builtin_amdgcn_sched_barrier(0);

  // The first D items behind them.
  u32x4* const ring = few_lds + wave * D * L::kUnits;
  const uint32_t oob = (uint32_t)(a.N / kTileN) * (uint32_t)a.G;   // a block past the weights
  int lu = u0, lg = wave;   // load cursor (wave-uniform)
  auto load_slot = [&](int j) __attribute__((always_inline)) {
    const bool in = lu < u1;
    const int ru = real_unit(lu);
    const int st0 = in ? (int)((uint32_t)ru % kPer) * S : 0;
    dma_issue<4, S>(ring + j * L::kUnits, rs, in ? (uint32_t)((uint32_t)ru / kPer) * (uint32_t)a.G + (uint32_t)lg : oob,
                    wbase + (uint32_t)st0 * 256u, lane);
    lg += W;
    if (lg >= a.G) {
      lg = wave;
      ++lu;
    }
  };
  if (nw) {
#pragma unroll
    for (int j = 0; j < D; ++j) load_slot(j);
  }
  // the codes have come: no wait for them inside the loop
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int h = 0; h < 2; ++h) asm volatile("" : "+v"(x[i][mb][h]));
  lds_barrier<true>();   // the scales are there

  f32x4 acc[MB][S];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < S; ++i) acc[mb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kJobs = MB * 4, kMine = (kJobs + W - 1) / W;   // (block, row of four) that a wave closes
  float gate[kMine][S];
#pragma unroll
  for (int k = 0; k < kMine; ++k)
#pragma unroll
    for (int i = 0; i < S; ++i) gate[k][i] = 0.f;

  int j = 0, left = T;   // slot of the next item, items not yet done
  for (int u = u0; u < u1; ++u) {
    const int ru = real_unit(u);
    const int st0 = (int)((uint32_t)ru % kPer) * S;
    static_for<0, NG>([&](auto ic) __attribute__((always_inline)) {
      constexpr int gi = decltype(ic)::value;
      if (gi >= nw) return;   // wave-uniform
      // this item has landed; the min(D - 1, left - 1) behind it may be in flight
      if (left >= D)
        wait_vm<(D - 1) * kL>();
      else
        wait_items<kL, D>(left - 1);
      RowsData<4, S, true> d;
      dma_read<4, S, true>(d, ring + j * L::kUnits, lane, st0);
      f32x4 sx[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        sx[mb] = *reinterpret_cast<const f32x4*>(sxl + (wave + W * gi) * 16 * MB + 16 * mb + 4 * q);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const uint32_t z = ((d.z >> (zsh + 4 * (st0 + i))) & 0xFu) * 0x01010101u;
        const float sw = bf16_bits_to_f32((d.s[i >> 1] >> (16 * (S == 1 ? (st0 & 1) : (i & 1)))) & 0xffffu);
        u32x4 lo, hi;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          lo[t] = a8_less(d.w[i][0][t] & 0x0F0F0F0Fu, z);
          hi[t] = a8_less((d.w[i][0][t] >> 4) & 0x0F0F0F0Fu, z);
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          i32x4 C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][0]),
                                                          __builtin_bit_cast(i32x4, lo), i32x4{0, 0, 0, 0}, 0, 0, 0);
          C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][1]),
                                                    __builtin_bit_cast(i32x4, hi), C, 0, 0, 0);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
            acc[mb][i][jj] = __builtin_fmaf((float)C[jj] * sw, sx[mb][jj], acc[mb][i][jj]);
        }
      }
      // the slot's reads have returned: load the item D ahead into it
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (left > D) load_slot(j);
      j = j + 1 == D ? 0 : j + 1;
      --left;
    });
    // Unit sums in wave order, row 4 q + jj of block mb by wave (4 mb + jj) % 8 (one block:
    // the halves of the workgroup take turns). With two buffers one barrier a unit: a buffer
    // is written again two barriers after it was read.
    const int n = u - u0, par = kBuf == 2 ? n & 1 : 0;
    if (kBuf == 1 && n) lds_barrier<true>();   // the unit before has been read
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < S; ++i) {
        red[wave][((par * MB + mb) * S + i) * 64 + lane] = acc[mb][i];
        acc[mb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    lds_barrier<true>();
    const int turn = kGlu ? n >> 1 : n;
    if (MB > 1 || (wave >> 2) == (turn & 1)) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int job = MB > 1 ? wave + W * k : wave & 3, mb = job >> 2, jj = job & 3;
        float v[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const int at = (((par * MB + mb) * S + i) * 64 + lane) * 4 + jj;
          v[i] = reinterpret_cast<const float*>(red[0])[at];
#pragma unroll
          for (int w = 1; w < W; ++w) v[i] += reinterpret_cast<const float*>(red[w])[at];
        }
        if (kGlu && (n & 1) == 0) {
#pragma unroll
          for (int i = 0; i < S; ++i) gate[k][i] = v[i];
        } else {
          const uint32_t ou = kGlu ? (uint32_t)u >> 1 : (uint32_t)u;   // output unit
          few_emit<OUT, S>(a, 16 * mb + 4 * q + jj, (int)(ou / kPer) * kTileN + 4 * c + (int)(ou % kPer) * S, v, gate[k]);
        }
      }
    }
  }
  wait_vm<0>();   // no load lands in LDS after the workgroup released it
}

template <int OUT, int S, int NG, int D, int MB>
bool launch(const FewArgs& f, hipStream_t st) {
  constexpr auto kern = &k_a8_few<OUT, S, NG, D, MB>;
  constexpr int red = kFewW * few_buffers<MB, S>() * MB * S * 1024;
  const int lds = kFewW * D * DmaSlot<4, S>::kUnits * 16 + f.a.G * 64 * MB;
  static_assert(kFewW * D * DmaSlot<4, S>::kUnits * 16 + kFewW * NG * 64 * MB + red <= kLdsBytes, "LDS of a CU");
  allow_lds<kern>(kFewW * D * DmaSlot<4, S>::kUnits * 16 + kFewW * NG * 64 * MB);
  kern<<<f.P, 64 * kFewW, lds, st>>>(f);
  return true;
}

template <int OUT, int S>
bool launch_few(const FewArgs& f, hipStream_t st) {
  const int ng = (f.a.G + kFewW - 1) / kFewW, M = f.a.M;
  if (M <= 16) {
    if (ng <= 3) return launch<OUT, S, 3, 3, 1>(f, st);
    if (ng <= 5) return launch<OUT, S, 5, 3, 1>(f, st);
    if (ng <= 8) return launch<OUT, S, 8, 3, 1>(f, st);
    if (ng <= 12) return launch<OUT, S, 12, 3, 1>(f, st);
    return ng <= 20 && launch<OUT, S, 20, 3, 1>(f, st);
  }
  if (M <= 32) {
    if (ng <= 5) return launch<OUT, S, 5, 3, 2>(f, st);
    return ng <= 10 && launch<OUT, S, 10, 3, 2>(f, st);
  }
  return M <= 64 && ng <= 5 && launch<OUT, S, 5, 3, 4>(f, st);
}

}  // namespace

// Launches the rows of `a` where this kernel takes them.
bool a8_few(int out, const A8Args& a, int cus, hipStream_t st) {
  if ((size_t)a.N * a.K / 2 >= (1ull << 32) || (size_t)a.M * a.K >= (1ull << 32)) return false;   // 32-bit offsets
  const int tiles = a.N / kTileN;
  const bool small = out != A8_GLU && 4 * tiles <= cus;   // 16-row units
  const int S = small ? 1 : 2;
  FewArgs f{a, 0, tiles * 4 / S};
  // as few workgroups as give none of them another unit
  const int n = out == A8_GLU ? f.U / 2 : f.U, most = (n + cus - 1) / cus;
  f.P = (n + most - 1) / most;
  if (out == A8_GLU) return launch_few<A8_GLU, 2>(f, st);
  if (out == A8_F32) return small ? launch_few<A8_F32, 1>(f, st) : launch_few<A8_F32, 2>(f, st);
  return small ? launch_few<A8_EPI, 1>(f, st) : launch_few<A8_EPI, 2>(f, st);
}

}  // namespace qw4
