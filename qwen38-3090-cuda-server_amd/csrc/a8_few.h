// Products of few rows in 8 bits (1 to 16, for shorter K up to 64, in one reading of the
// weights): qw4_a8_linear's decode, verify and small batches. HBM-bound: one / 9 / 16 / 32
// rows of 34816 x 5120 gated 17.9 / 19.6 / 20.3 / 24.8 us (93 MB: 5.2 TB/s of one row), 9 of
// 248320 x 5120 in fp32 105.8 (6.3 TB/s), 48 156; of small weights the launch and the first loads:
// one row of 5120 x 4096 5.1 us.
//
// Workgroup p owns whole units (S row quads of a tile, 16 or 32 weight rows, over all of
// K); wave w takes the groups w, w + W, ... and the units are summed over the waves in
// wave order, as in the bf16 kernel for few rows. A wave meets the same groups in every
// unit, so it keeps their codes: 8 registers a group and 16 rows, half of bf16's, and in
// the order that the nibbles of a weight word have, so that they are MFMA operands as
// they lie in memory. Weights stream past them through LDS-DMA slots, D items (a group of
// a unit) ahead, across units; the codes come with the items of the first unit.
//
// An item's nibbles are int8 operands as they are, and the zero point comes off the sums:
// sum (q - z) x = sum q x - z X, X the sum of the row's codes, exactly in int32. X and the
// rows' scales lie in LDS. Three vector instructions a word instead of seven.
//
// Row r of a block is MFMA row 4 (r % 4) + r / 4, so that up to 4 rows take one result
// register of four, up to 8 two (JJ): what scales the sums is as much as the rows need (one
// row of 5120 x 17408 11.6 us, with four registers 13.1; 8 rows of 34816 x 5120 19.1 and 19.8).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "a8.h"
#include "skinny.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

// Buffers of the waves' sums of a part.
template <int MB, int S>
constexpr int few_buffers(int W) { return MB * S * W <= 16 ? 2 : 1; }
// 16-byte units that they take for a wave, and its codes of 16 rows and a group.
template <int MB, int S, int JJ>
constexpr int few_red(int W) {
  const int sums = few_buffers<MB, S>(W) * MB * S * 16 * JJ;
  return JJ > 1 && sums < 128 ? 128 : sums;
}

// Row m, columns n0 + i: the sums (gate, up) of a unit.
template <int OUT, int S>
__device__ __forceinline__ void few_emit(const A8Args& a, int m, int n0, float (&v)[OUT == A8_GLU ? 2 : 1][S]) {
  if (m >= a.M) return;
  const size_t at = (size_t)m * a.ld + n0;
  if constexpr (OUT == A8_F32) {
    float* y = static_cast<float*>(a.y) + at;
#pragma unroll
    for (int i = 0; i < S; ++i) y[i] = v[0][i];
  } else {
    constexpr bool kGlu = OUT == A8_GLU;
    float b[S], r[S];
#pragma unroll
    for (int j = 0; j < (kGlu ? 2 : 1); ++j) {
      load_cols<S>(b, a.epi.bias, (size_t)n0 + j * a.epi.up);
#pragma unroll
      for (int i = 0; i < S; ++i) v[j][i] += b[i];
    }
    load_cols<S>(r, a.epi.res, at);
    epilogue_act<kGlu, S>(v, a.epi.act);
    uint16_t* y = static_cast<uint16_t*>(a.y) + at;
    if constexpr (S == 1) {
      y[0] = to_bf16(v[0][0] + r[0]);
    } else {
#pragma unroll
      for (int i = 0; i < S / 2; ++i)
        reinterpret_cast<uint32_t*>(y)[i] = pack_bf16x2(v[0][2 * i] + r[2 * i], v[0][2 * i + 1] + r[2 * i + 1]);
    }
  }
}

struct FewArgs {
  A8Args a;
  int P, U;
};

template <int OUT, int S, int NG, int W, int D, int MB, int JJ>
__global__ __launch_bounds__(64 * W, W / 4) void k_a8_few(FewArgs f) {
  using L = DmaSlot<4, S>;
  typedef float fJ __attribute__((ext_vector_type(JJ)));
  constexpr int PT = OUT == A8_GLU ? 2 : 1;   // parts of a unit: gate and up
  constexpr int kL = PT * L::kLoads, kLX = kL + 2 * MB, kSlot = PT * L::kUnits, kBuf = few_buffers<MB, S>(W);
  constexpr int kPer = 4 / S;
  const A8Args& a = f.a;
  // A wave's sums of a part; before it has any, its codes of a group on their way into MFMA rows.
  constexpr int kRed = few_red<MB, S, JJ>(W);
  __shared__ u32x4 room[W][kRed];
  extern __shared__ u32x4 few_lds[];   // the waves' slots; scales and code sums [G][2][16 MB]
  float* const sxl = reinterpret_cast<float*>(few_lds + W * D * kSlot);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4;
  SkinnyRsrc rs;
  rs.qw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(a.qw), 0, (int)((uint32_t)(a.N / kTileN) * a.G * 4096u),
                                            0x00020000);
  rs.sc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.sc), 0,
                                            (int)((uint32_t)(a.N / kTileN) * a.G * (uint32_t)kMetaBytes), 0x00020000);
  rs.x = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.q), 0, (int)((uint32_t)a.M * (uint32_t)a.K), 0x00020000);
  const uint32_t wbase = Fmt<4>::woff(q, c), up = (uint32_t)(a.epi.up / kTileN) * (uint32_t)a.G;
  const int p = blockIdx.x;
  const int u0 = (int)((long long)p * f.U / f.P), u1 = (int)((long long)(p + 1) * f.U / f.P);
  const int nw = wave < a.G ? (a.G - 1 - wave) / W + 1 : 0;   // groups of this wave (<= NG)

  // Scales: of MFMA row m of block b, at 16 b + m.
  for (int i = threadIdx.x; i < a.G * 16 * MB; i += 64 * W) {
    const int g = i / (16 * MB), m = i - g * (16 * MB), row = (m & ~15) + 4 * (m & 3) + ((m & 15) >> 2);
    sxl[(2 * g) * 16 * MB + m] = row < a.M ? a.scale[(size_t)g * a.max_rows + row] : 0.f;
  }

  u32x4 x[NG][MB][2];
  // Codes of the wave's group i; rows past M are zeros without traffic. Up to 4 rows: row
  // 4 (c % 4) + c / 4, chunk q, as MFMA takes them. More: whole 128-byte rows, 8 a load, which
  // pass through LDS; as MFMA takes them, each lane of a load would be a line of its own
  // (down of 16 rows 17.7 us, 15.9 so; of one row 11.6 and 12.6).
  constexpr bool kDirect = JJ == 1;
  const uint32_t xbase = kDirect ? (uint32_t)(4 * (c & 3) + (c >> 2)) * (uint32_t)a.K + 32u * q
                                 : (uint32_t)(lane >> 3) * (uint32_t)a.K + 16u * (lane & 7);
  const uint32_t xmb = 16u * (uint32_t)a.K, xh = kDirect ? 16u : 8u * (uint32_t)a.K;
  auto load_codes = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        x[i][mb][h] = __builtin_amdgcn_raw_buffer_load_b128(
            rs.x, xbase + mb * xmb + h * xh, (uint32_t)(wave + W * i) * 128u, 0);
  };
  u32x4* const ring = few_lds + wave * D * kSlot;
  // load cursor (wave-uniform): group, unit, block and row quad of the next item; a block past
  // the weights once there is none
  const uint32_t past = (uint32_t)(a.N / kTileN) * (uint32_t)a.G;
  int lg = wave, lu = u0;
  uint32_t lblk = (uint32_t)(u0 / kPer) * (uint32_t)a.G + (uint32_t)wave, lst = (uint32_t)(u0 % kPer) * S * 256u;
  auto load_slot = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < PT; ++t)
      dma_issue<4, S>(ring + j * kSlot + t * L::kUnits, rs, lblk + t * up, wbase + lst, lane);
    lg += W;
    lblk += W;
    if (lg >= a.G) {
      lg = wave;
      ++lu;
      lblk = lu < u1 ? (uint32_t)(lu / kPer) * (uint32_t)a.G + (uint32_t)wave : past;
      lst = (uint32_t)(lu % kPer) * S * 256u;
    }
  };
  if (nw) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (j < NG) load_codes(j < NG ? j : 0);
      load_slot(j);
    }
  }
  lds_barrier<true>();   // the scales are there

  const i32x4 start = {kA8Start, kA8Start, kA8Start, kA8Start};
  fJ acc[PT][MB][S];
#pragma unroll
  for (int t = 0; t < PT; ++t)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < S; ++i) acc[t][mb][i] = fJ{};
  constexpr int kJobs = MB * JJ, kMine = (kJobs + W - 1) / W;   // (block, result register) that a wave closes

  int j = 0, left = nw * (u1 - u0);   // slot of the next item, items not yet done
  auto unit = [&](int u, auto first) __attribute__((always_inline)) {
    constexpr bool kFirst = decltype(first)::value;
    const int st0 = (u % kPer) * S, zsh = 16 * (c & 1) + 4 * st0;
    static_for<0, NG>([&](auto ic) __attribute__((always_inline)) {
      constexpr int gi = decltype(ic)::value;
      if (gi >= nw) return;   // wave-uniform
      // this item has landed; the min(D - 1, left - 1) behind it may be in flight (of the
      // first unit, with their codes)
      if (kFirst && gi + D <= nw)
        wait_vm<(D - 1) * kLX>();
      else if (left >= D)
        wait_vm<(D - 1) * kL>();
      else
        wait_items<kL, D>(left - 1);
      RowsData<4, S, true> d[PT];
#pragma unroll
      for (int t = 0; t < PT; ++t) dma_read<4, S, true>(d[t], ring + j * kSlot + t * L::kUnits, lane, st0);
      if constexpr (kFirst && !kDirect) {   // through LDS: chunk k of row m at k ^ g(m), as in the tiles
        auto at = [](int m, int k) { return m * 8 + (k ^ (m & 7) ^ ((m >> 3) & 1)); };
        u32x4* const own = room[wave];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
          for (int h = 0; h < 2; ++h) own[at(8 * h + (lane >> 3), lane & 7)] = x[gi][mb][h];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int h = 0; h < 2; ++h) x[gi][mb][h] = own[at(4 * (c & 3) + (c >> 2), 2 * q + h)];
          __builtin_amdgcn_wave_barrier();
        }
      }
      float* const sg = sxl + 2 * (wave + W * gi) * 16 * MB + 4 * q;
      fJ sx[MB], xs[MB];   // scales, minus the sums of the rows' codes
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        sx[mb] = *reinterpret_cast<const fJ*>(sg + 16 * mb);
        if constexpr (kFirst) {   // the same in all columns
          const i32x4 minus = {-1, -1, -1, -1};
          i32x4 C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][0]), minus, i32x4{0, 0, 0, 0}, 0, 0, 0);
          C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][1]), minus, C, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < JJ; ++k) xs[mb][k] = __int_as_float(C[k]);
          if (c == 0) *reinterpret_cast<fJ*>(sg + 16 * MB + 16 * mb) = xs[mb];
        } else {
          xs[mb] = *reinterpret_cast<const fJ*>(sg + 16 * MB + 16 * mb);
        }
      }
#pragma unroll
      for (int t = 0; t < PT; ++t) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const int z = (int)((d[t].z >> (zsh + 4 * i)) & 0xFu);
          const float sw = bf16_bits_to_f32((d[t].s[i >> 1] >> (16 * (S == 1 ? (st0 & 1) : (i & 1)))) & 0xffffu);
          const float less = -kA8Magic * sw;
          u32x4 lo, hi;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            lo[k] = d[t].w[i][0][k] & 0x0F0F0F0Fu;
            hi[k] = (d[t].w[i][0][k] >> 4) & 0x0F0F0F0Fu;
          }
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            i32x4 C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][0]),
                                                            __builtin_bit_cast(i32x4, lo), start, 0, 0, 0);
            C = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x[gi][mb][1]),
                                                      __builtin_bit_cast(i32x4, hi), C, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < JJ; ++k) {
              const int v = __mul24(z, __float_as_int(xs[mb][k])) + C[k];
              const float p = __builtin_fmaf(__int_as_float(v), sw, less);
              acc[t][mb][i][k] = __builtin_fmaf(p, sx[mb][k], acc[t][mb][i][k]);
            }
          }
        }
      }
      // the slot's reads have returned: load the item D ahead into it
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (kFirst && gi + D < NG && gi + D < nw) load_codes(gi + D < NG ? gi + D : 0);
      if (left > D) load_slot(j);
      j = j + 1 == D ? 0 : j + 1;
      --left;
    });
    // A part's sums in wave order, register k of block mb by wave (JJ mb + k) % W (one block:
    // JJ waves at a time take turns). With two buffers one barrier a part: a buffer is
    // written again two barriers after it was read.
    const int n = u - u0, turn = n % (W / JJ);
    const bool closes = MB > 1 || wave / JJ == turn;
    float v[kMine][PT][S];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      const int par = kBuf == 2 ? (n * PT + t) & 1 : 0;
      if (kBuf == 1 && n + t) lds_barrier<true>();   // the part before has been read
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < S; ++i) {
          reinterpret_cast<fJ*>(room[wave])[((par * MB + mb) * S + i) * 64 + lane] = acc[t][mb][i];
          acc[t][mb][i] = fJ{};
        }
      lds_barrier<true>();
      if (closes) {
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const int job = MB > 1 ? wave + W * k : wave % JJ, mb = job / JJ, jj = job % JJ;
          if (kJobs % W && MB > 1 && job >= kJobs) break;
#pragma unroll
          for (int i = 0; i < S; ++i) {
            const int at = (((par * MB + mb) * S + i) * 64 + lane) * JJ + jj;
            float r = reinterpret_cast<const float*>(room[0])[at];
#pragma unroll
            for (int w = 1; w < W; ++w) r += reinterpret_cast<const float*>(room[w])[at];
            v[k][t][i] = r;
          }
        }
      }
    }
    if (closes) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int job = MB > 1 ? wave + W * k : wave % JJ, mb = job / JJ, jj = job % JJ;
        if (kJobs % W && MB > 1 && job >= kJobs) break;
        few_emit<OUT, S>(a, 16 * mb + 4 * jj + q, (u / kPer) * kTileN + 4 * c + st0, v[k]);
      }
    }
  };
  unit(u0, std::true_type{});
  for (int u = u0 + 1; u < u1; ++u) unit(u, std::false_type{});
  wait_vm<0>();   // no load lands in LDS after the workgroup released it
}

template <int OUT, int S, int NG, int W, int D, int MB, int JJ>
bool launch(const FewArgs& f, hipStream_t st) {
  constexpr auto kern = &k_a8_few<OUT, S, NG, W, D, MB, JJ>;
  constexpr int slots = (OUT == A8_GLU ? 2 : 1) * W * D * DmaSlot<4, S>::kUnits * 16;
  constexpr int fixed = W * few_red<MB, S, JJ>(W) * 16;
  static_assert(slots + W * NG * 128 * MB + fixed <= kLdsBytes, "LDS of a CU");
  allow_lds<kern>(slots + W * NG * 128 * MB);
  kern<<<f.P, 64 * W, slots + f.a.G * 128 * MB, st>>>(f);
  return true;
}

// Items in flight a wave: gated ones are twice as long.
template <int OUT, int S, int JJ>
bool launch16(const FewArgs& f, hipStream_t st) {
  constexpr int D = OUT == A8_GLU ? 2 : 3;
  const int G = f.a.G;
  // one unit a workgroup and a long K: 16 waves (5120 x 17408, one / 9 rows 11.6 / 14.1 us, in 8
  // waves 15.6 / 17.8)
  if constexpr (OUT != A8_GLU) {
    if (G > 64 && f.P >= f.U) {
      if (G <= 80) return launch<OUT, S, 5, 16, 2, 1, JJ>(f, st);
      if (G <= 144) return launch<OUT, S, 9, 16, 2, 1, JJ>(f, st);
    }
  }
  if (G <= 24) return launch<OUT, S, 3, 8, D, 1, JJ>(f, st);
  if (G <= 40) return launch<OUT, S, 5, 8, D, 1, JJ>(f, st);
  if (G <= 64) return launch<OUT, S, 8, 8, D, 1, JJ>(f, st);
  return G <= 160 && launch<OUT, S, 20, 8, D, 1, JJ>(f, st);
}

// More than 32 rows in gated units of 16 rows each: those of 32 have twice the sums, which do
// not fit the registers beside the codes (48 rows of 34816 x 5120 30.3 and 44.8 us).
template <int OUT, int S>
bool launch_few(const FewArgs& f, hipStream_t st) {
  constexpr int D = OUT == A8_GLU ? 2 : 3;
  const int G = f.a.G, M = f.a.M;
  if constexpr (OUT != A8_GLU || S == 1) {
    // 48 rows of 7168 x 5120 12.8 us, as tiles 15.7, of 5120 x 4096 10.3 and 12.4, of 34816 x 5120
    // gated 30.3 and 36.7; 64 of 5120 x 2048 9.1 and 10.0, but of 5120 x 4096 14.7 and 12.7, and
    // with more units than workgroups, of 34816 x 2048 gated, 21.6 and 19.0
    if (M > 48) return G <= 24 && f.P >= f.U && launch<OUT, S, 3, 8, D, 4, 4>(f, st);
    if (M > 32) return G <= 40 && launch<OUT, S, 5, 8, D, 3, 4>(f, st);
  }
  if constexpr (OUT != A8_GLU || S == 2) {
    if (M <= 4) return launch16<OUT, S, 1>(f, st);
    if (M <= 8) return launch16<OUT, S, 2>(f, st);
    if (M <= 16) return launch16<OUT, S, 4>(f, st);
    if (G <= 40) return launch<OUT, S, 5, 8, D, 2, 4>(f, st);
    // gated, codes of more than 8 groups a wave do not fit beside the sums: 32 rows of 34816 x 8192
    // 34.2 us, as tiles 39.9, with spills 43.9; of 28672 x 10240 as tiles 36.6, with spills 41.6.
    // Of few columns tiles in slices are the faster: 4096 x 8192 12.8 and 15.5
    if constexpr (OUT == A8_GLU)
      return G <= 64 && launch<OUT, S, 8, 8, D, 2, 4>(f, st);
    else
      return G <= 80 && launch<OUT, S, 10, 8, D, 2, 4>(f, st);
  }
  return false;
}

}  // namespace
}  // namespace qw4
