// k_grouped_rows: the products grouped by expert where experts have few rows (a decoded
// token, a verify block, a short prompt), for K up to 8 x kMaxGroups groups.
//
// Bound by the chosen experts' weights, each of which a call reads once. The split and
// the sums are k_rows_xr's (rows_xr.hip): blocks of 16 MB rows of an expert against units
// of S row quads of its weight over all of K -- gated, half of them gate quads and half
// the up quads of the same columns, so that a lane has both sums of a column and a unit
// is half as wide; workgroup p owns a run of units, wave w the groups w, w + 8, ...; the
// block's activations sit in registers while the weights stream through LDS slots, D
// items ahead, across units, blocks and experts; the waves' sums meet in LDS in wave
// order. Weights are used exactly: 128 + q as a bf16 operand, scale and zero point in
// fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/qwen_w4a16.h"
#include "grouped.h"
#include "skinny.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

constexpr int kW = 8;           // waves
constexpr int kMaxGroups = 8;   // groups a wave can hold

// A place in the run of (block, unit): the block, its expert and the unit in it.
struct Place {
  int block, unit, e;
};

// Item slot (16-byte units): S x 64 weight chunks, then a 256-byte area for each scale
// and zero-point record (gated: the gate tile's and the up tile's).
template <bool GLU, int S>
struct ItemSlot {
  static constexpr int kRecords = GLU ? 2 : 1;
  static constexpr int kQuads = S / kRecords;   // quads of a record
  static constexpr int kUnits = S * 64 + kRecords * 16;
  static constexpr int kLoads = S + kRecords;
};

template <bool GLU, int S, int NG, int D, int MB>
__global__ __launch_bounds__(64 * kW) void k_grouped_rows(GroupedArgs a) {
  using L = ItemSlot<GLU, S>;
  constexpr int kL = L::kLoads, Q = L::kQuads;
  constexpr uint32_t kPer = 4 / Q;         // units of a weight tile
  constexpr int kArea = 2 * MB * S * 64;   // a wave's sums of a unit, two buffers
  constexpr int kSums = MB == 1 ? 0 : NG * MB * 4;   // MB > 1: a wave's row sums (no registers left)
  // One LDS object: of several the compiler tells the accesses apart and waits for every
  // load into the slots before it reads the sums (vmcnt(0) in place of the counted waits).
  __shared__ u32x4 lds[kW * (D * L::kUnits + kArea + kSums) + (kMaxExperts + 1 + kW + 3) / 4];
  static_assert(sizeof(lds) <= kLdsBytes, "the CU's LDS");
  u32x4* const slots = lds;
  f32x4* const red = reinterpret_cast<f32x4*>(slots + kW * D * L::kUnits);
  f32x4* const csum = red + kW * kArea;
  int* const start = reinterpret_cast<int*>(csum + kW * kSums);
  int* const wsum = start + kMaxExperts + 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4;
  // Blocks before each expert: up to 64 experts a lane each, without LDS and its barriers
  // (every wave for itself: one token through 8 of 64 experts, 2048 -> 2 x 1024 / 1024 -> 2048,
  // 7.3 / 6.3 -> 6.1 / 5.2 us); else expert_starts.
  auto blocks_of = [](int rows, int) { return (rows + 16 * MB - 1) / (16 * MB); };
  const bool in_lanes = a.E <= 64;
  int all[1], my_lo = 0, my_hi = 0, my_start = 0;
  if (in_lanes) {
    if (lane < a.E) expert_rows(a, lane, my_lo, my_hi);
    const int mine = blocks_of(my_hi - my_lo, 0);
    int run = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(run, off, 64);
      if (lane >= off) run += v;
    }
    my_start = lane < a.E ? run - mine : 0x7fffffff;
    all[0] = __builtin_amdgcn_readlane(run, 63);
  } else {
    expert_starts<64 * kW>(a, start, wsum, all, blocks_of);
  }
  auto start_of = [&](int e) __attribute__((always_inline)) {
    return in_lanes ? __builtin_amdgcn_readlane(my_start, e) : __builtin_amdgcn_readfirstlane(start[e]);
  };
  // units of a block, and this workgroup's run of them
  const int per = a.ld / (16 * Q);
  const long long total = (long long)all[0] * per;
  const int p = blockIdx.x;
  const long long u0 = p * total / a.P, u1 = (p + 1) * total / a.P;
  int left_units = (int)(u1 - u0);
  if (left_units <= 0) return;
  const int nw = wave < a.G ? (a.G - 1 - wave) / kW + 1 : 0;   // groups of this wave (<= NG)
  int left = nw * left_units;                                   // items not yet done

  // a place moves on to the next unit, block and expert
  auto begin = [&](Place& v) __attribute__((always_inline)) {
    v.block = (int)(u0 / per);
    v.unit = (int)(u0 - (long long)v.block * per);
    // the last expert that starts at or before the block (see expert_of)
    v.e = in_lanes ? (int)__popcll(__ballot(my_start <= v.block)) - 1 : expert_of(start, a.E, 1, v.block);
  };
  auto next = [&](Place& v) __attribute__((always_inline)) {
    if (++v.unit == per) {
      v.unit = 0;
      ++v.block;
      while (v.e + 1 < a.E && start_of(v.e + 1) <= v.block) ++v.e;
    }
  };

  // The load cursor: the unit's place, its group as byte offsets into the expert's
  // weights and scales, and the lanes' offsets. A wave has only one other on its SIMD, so
  // its scalar work is not hidden: what an item needs is kept up to date by additions.
  Place lp;
  begin(lp);
  int lg = wave, lunits = left_units;
  __amdgpu_buffer_rsrc_t lqw, lsc;
  const uint32_t blocks = (uint32_t)(a.n / kTileN) * (uint32_t)a.G;   // weight blocks of an expert
  const uint32_t up_blocks = (uint32_t)(a.epi.up / kTileN) * (uint32_t)a.G;
  const uint32_t wbase = Fmt<4>::woff(q, c);
  uint32_t wsoff = 0, msoff = 0;
  uint32_t wvoff = 0;
  const uint32_t mvoff = lane < 40 ? (uint32_t)lane * 4u : 0u;
  auto weights = [&]() __attribute__((always_inline)) {
    const size_t blk = (size_t)lp.e * blocks;
    lqw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(a.qw + blk * kWordsPerBlock), 0,
                                            (int)(blocks * 4096u), 0x00020000);
    lsc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.sc + blk * kMetaU16), 0,
                                            (int)(blocks * (uint32_t)kMetaBytes), 0x00020000);
  };
  auto unit = [&]() __attribute__((always_inline)) {
    const uint32_t ru = (uint32_t)lp.unit, blk = ru / kPer * (uint32_t)a.G + (uint32_t)wave;
    wsoff = (uint32_t)__builtin_amdgcn_readfirstlane(blk * 4096u);
    msoff = (uint32_t)__builtin_amdgcn_readfirstlane(blk * (uint32_t)kMetaBytes);
    wvoff = wbase + ru % kPer * Q * 256u;
  };
  weights();
  unit();
  u32x4* const ring = slots + wave * D * L::kUnits;
  auto load_slot = [&](int j) __attribute__((always_inline)) {
    u32x4* const slot = ring + j * L::kUnits;
#pragma unroll
    for (int h = 0; h < L::kRecords; ++h) {
#pragma unroll
      for (int i = 0; i < Q; ++i)
        dma_load16(lqw, slot + (h * Q + i) * 64, wvoff + i * 256u, wsoff + h * (up_blocks * 4096u));
      dma_load4(lsc, slot + S * 64 + h * 16, mvoff, msoff + h * (up_blocks * (uint32_t)kMetaBytes));
    }
    wsoff = (uint32_t)__builtin_amdgcn_readfirstlane(wsoff + kW * 4096u);
    msoff = (uint32_t)__builtin_amdgcn_readfirstlane(msoff + kW * (uint32_t)kMetaBytes);
    lg += kW;
    if (lg < a.G) return;
    lg = wave;
    if (--lunits > 0) {
      const int e = lp.e;
      next(lp);
      if (lp.e != e) weights();
      unit();
    }
  };
  if (nw > 0) {
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (j < left) load_slot(j);
  }

  const NibConst k = nib_const();
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u,
                                                       0x3F803F80u, 0x3F803F80u});
  u32x4 x[NG][MB][4];
  f32x4 Cs[MB == 1 ? NG : 1];
  Place at;
  begin(at);
  int m0 = 0, rows = 0;   // the block's first position and rows
  // The block's activations in MFMA operand order: lane c + 16 q holds row c, chunks 4 q
  // .. 4 q + 3 of each of the wave's groups, and their sums over the group.
  auto load_x = [&]() __attribute__((always_inline)) {
    int lo, hi;
    if (in_lanes) {
      lo = __builtin_amdgcn_readlane(my_lo, at.e);
      hi = __builtin_amdgcn_readlane(my_hi, at.e);
    } else {
      expert_rows(a, at.e, lo, hi);
      lo = __builtin_amdgcn_readfirstlane(lo);
      hi = __builtin_amdgcn_readfirstlane(hi);
    }
    const int nth = at.block - start_of(at.e);   // < 0: offsets of no plan
    m0 = lo + nth * 16 * MB;
    rows = nth < 0 ? 0 : min(hi - m0, 16 * MB);
    const uint32_t row_bytes = (uint32_t)a.K * 2u;
    const uint16_t* x0 = a.tokens ? a.x : a.x + (size_t)m0 * a.K;
    const uint32_t bytes = a.tokens ? a.x_bytes : (uint32_t)max(rows, 0) * row_bytes;
    const __amdgpu_buffer_rsrc_t rx =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(x0), 0, (int)bytes, 0x00020000);
    uint32_t off[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int m = 16 * mb + c;
      const int row = m >= rows ? -1 : a.tokens ? a.tokens[m0 + m] : m;
      const uint64_t o = (uint64_t)(uint32_t)row * row_bytes;
      off[mb] = o < bytes ? (uint32_t)o + (uint32_t)q * 64u : bytes;   // past x: zeros
    }
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          x[i][mb][t] = u32x4{0u, 0u, 0u, 0u};
          if (i < nw)
            x[i][mb][t] = __builtin_amdgcn_raw_buffer_load_b128(rx, off[mb] + t * 16u,
                                                                (uint32_t)(wave + kW * i) * 256u, 0);
        }
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        f32x4 cs;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          cs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, x[i][mb][t]), ones,
              t == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : cs, 0, 0, 0);
        if (MB == 1)
          Cs[MB == 1 ? i : 0] = cs;
        else if (c == 0)   // the same for all 16 columns; read by this wave alone
          csum[wave * kSums + (i * MB + mb) * 4 + q] = cs;
      }
  };
  load_x();

  f32x4 acc[MB][S];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < S; ++i) acc[mb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  int j = 0, n = 0;   // slot of the next item; units closed
  while (true) {
    const int st0 = (int)((uint32_t)at.unit % kPer) * Q;
    static_for<0, NG>([&](auto ic) __attribute__((always_inline)) {
      constexpr int gi = decltype(ic)::value;
      if (gi >= nw) return;   // wave-uniform
      // this item has landed; the min(D - 1, left - 1) behind it may be in flight
      if (left >= D)
        wait_vm<(D - 1) * kL>();
      else
        wait_items<kL, D>(left - 1);
      const u32x4* const slot = ring + j * L::kUnits;
      u32x4 w[S];
      float sf[S], zf[S];
#pragma unroll
      for (int i = 0; i < S; ++i) w[i] = slot[i * 64 + lane];
#pragma unroll
      for (int h = 0; h < L::kRecords; ++h) {
        const uint32_t* const rec = reinterpret_cast<const uint32_t*>(slot + S * 64 + h * 16);
        const uint32_t z = rec[32 + (c >> 1)] >> (16 * (c & 1) + 4 * st0);
#pragma unroll
        for (int i = 0; i < Q; ++i) {   // row 4 c + st0 + i
          const uint32_t s2 = rec[(4 * c + st0 + i) >> 1];
          sf[h * Q + i] = bf16_bits_to_f32((s2 >> (16 * (Q == 1 ? st0 & 1 : i & 1))) & 0xffffu);
          zf[h * Q + i] = 128.0f + (float)((z >> (4 * i)) & 0xFu);
        }
      }
      f32x4 C[MB][S];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const bf16x8 B = nib8(w[i][t], k);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            C[mb][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, x[gi][mb][t]), B,
                t == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : C[mb][i], 0, 0, 0);
        }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const f32x4 cs = MB == 1 ? Cs[MB == 1 ? gi : 0] : csum[wave * kSums + (gi * MB + mb) * 4 + q];
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) acc[mb][i][jj] += sf[i] * (C[mb][i][jj] - zf[i] * cs[jj]);
      }
      // the slot's reads have returned: load the item D ahead into it
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (left > D) load_slot(j);
      j = j + 1 == D ? 0 : j + 1;
      --left;
    });
    // Unit sums in wave order; row 4 q + jj by wave jj (mod 4) of one half of the
    // workgroup, the halves taking turns (MB = 2: a half each row block). Two buffers, one
    // barrier a unit: a buffer is written again two barriers after it was read.
    const int par = n & 1;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < S; ++i) {
        red[wave * kArea + ((par * MB + mb) * S + i) * 64 + lane] = acc[mb][i];
        acc[mb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    lds_barrier<true>();
    if (MB == 2 || (wave >> 2) == (n & 1)) {
      const int jj = wave & 3, mb = MB == 2 ? wave >> 2 : 0;
      const int m = 16 * mb + 4 * q + jj;
      const int n0 = (int)((uint32_t)at.unit / kPer) * kTileN + 4 * c + st0;
      float f[L::kRecords][Q];
#pragma unroll
      for (int h = 0; h < L::kRecords; ++h) {
        float b[Q];
        load_cols<Q>(b, a.epi.bias, (size_t)at.e * a.n + h * a.epi.up + n0);
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const int from = (((par * MB + mb) * S + h * Q + i) * 64 + lane) * 4 + jj;
          float v = reinterpret_cast<const float*>(red)[from];
#pragma unroll
          for (int w = 1; w < kW; ++w) v += reinterpret_cast<const float*>(red + w * kArea)[from];
          f[h][i] = v + b[i];
        }
      }
      epilogue_act<GLU, Q>(f, a.epi.act);
      if (m < rows) {
        const size_t to = (size_t)(m0 + m) * a.ld + n0;
        if constexpr (Q == 1) {
          a.y[to] = to_bf16(f[0][0]);
        } else {
#pragma unroll
          for (int i = 0; i < Q / 2; ++i)
            reinterpret_cast<uint32_t*>(a.y + to)[i] = pack_bf16x2(f[0][2 * i], f[0][2 * i + 1]);
        }
      }
    }
    ++n;
    if (--left_units == 0) break;
    const int block = at.block;
    next(at);
    if (at.block != block) load_x();
  }
  wait_vm<0>();   // no load lands in LDS after the workgroup released it
}

template <bool GLU, int S, int NG, int D, int MB>
void launch(const GroupedArgs& a, hipStream_t st) {
  k_grouped_rows<GLU, S, NG, D, MB><<<a.P, 64 * kW, 0, st>>>(a);
}

// Registers for 2, 5 or 8 groups a wave (K up to 2048, 5120, 8192).
template <bool GLU, int S, int D>
void launch_ng(const GroupedArgs& a, hipStream_t st) {
  const int ng = (a.G + kW - 1) / kW;
  if (ng <= 2)
    launch<GLU, S, 2, D, 1>(a, st);
  else if (ng <= 5)
    launch<GLU, S, 5, D, 1>(a, st);
  else
    launch<GLU, S, kMaxGroups, D, 1>(a, st);
}

template <bool GLU>
void launch_rows(const GroupedArgs& a, int MB, int S, hipStream_t st) {
  if (MB == 2)
    launch<GLU, 2, 5, 4, 2>(a, st);
  else if (S == 4)
    launch_ng<GLU, 4, 2>(a, st);
  else
    launch_ng<GLU, 2, 3>(a, st);
}

// What the estimates below share: E experts, mean rows of each, experts in use (a token's
// are different ones; many tokens' as if drawn evenly).
struct Shares {
  double E, mean, used;
  explicit Shares(const GroupedArgs& a) : E(a.E), mean((double)a.R / a.E) {
    used = 4 * (long long)a.R <= a.E ? a.R : E * (1.0 - std::exp(-mean));
  }
  // Blocks of h rows: R rows in random shares make E (R / (E h) + 1/2).
  double blocks(int h) const { return std::max(used, mean < 1 ? 0. : E * (mean / h + 0.5)); }
};

// us of blocks of h rows in units of S row quads: a unit of the fullest workgroup costs its
// groups and its close.
double rows_us(const GroupedArgs& a, const Shares& sh, bool glu, int cus, int h, int S) {
  const int ng = (a.G + kW - 1) / kW;
  const double units = std::max(1., std::ceil(sh.blocks(h) * (a.ld / (16 * (glu ? S / 2 : S))) / cus));
  return h == 16 ? 6 + units * (0.15 + 0.31 * S * ng) : 24 + units * (0.6 + 0.7 * ng);
}

// us of tiles of h rows, two a CU at once: a round costs its groups, by the share of the
// rows in use (ending tiles start at a half), and its start and store; the weights are read
// before they compute.
double tiles_us(const GroupedArgs& a, const Shares& sh, int cus, int h) {
  const double bytes = sh.used * a.n * a.G * (64 + 2.5);
  const double rounds = std::max(1., sh.blocks(h) * a.tiles_n / (2. * cus));
  const double share = std::min(1., std::max(0.5, sh.mean / 32));
  return bytes / 5.4e6 + rounds * (h == 128 ? 15 + 1.7 * share * a.G : 14 + 0.95 * share * a.G);
}

}  // namespace

// The estimated fastest, as qw4_tune_grouped numbers them (3 for tiles of 256 rows too): blocks
// of 16 rows, blocks of 32 (4 and 5 groups a wave: fewer do not pay, more do not fit the
// registers), tiles of 128 rows or of 64. Fitted over 350 shapes (4 to 128 experts, K of 256 to
// 8192, 192 to 5120 weight rows, 3 to 200 rows an expert); over 400 others 2.0% in the geometric
// mean from the fastest. By the mean rows of an expert alone (40, or 24 with long K) and without
// the tiles of 64 rows it was 10%, and up to six times where tiles are few. us, blocks of 16 / of
// 32 / tiles of 128 / of 64; experts, K -> weight rows, rows an expert:
//   32, 5120 -> 4352 gated   25 rows  129 / 119 / 165 / 121,    38  169 / 142 / 164 / 126
//   64, 2048 -> 2048 gated   25       54 / 56 / 50 / 56,        50  90 / 82 / 76 / 59
//   32, 2176 -> 5120         25       73 / 73 / 74 / 58,        125  287 / 214 / 117 / 134
//   64, 1024 -> 2048         32       38 / 45 / 45 / -,         48  52 / 58 / 45 / -
//   16, 6144 -> 2048 gated   32       52 / - / 89 / -
//    4, 7808 -> 320          50       18 / - / 108 / -
int grouped_form(const GroupedArgs& a, bool glu, int cus, bool exact) {
  const Shares sh(a);
  const int ng = (a.G + kW - 1) / kW;
  const bool tiles = !exact || ng > kMaxGroups;
  int form = 3;
  double best = tiles ? tiles_us(a, sh, cus, 128) : HUGE_VAL;
  auto consider = [&](int f, double us) {
    if (us < best) {
      best = us;
      form = f;
    }
  };
  if (tiles) consider(5, tiles_us(a, sh, cus, 64));
  if (ng == 4 || ng == 5) consider(2, rows_us(a, sh, glu, cus, 32, 2));
  if (ng <= kMaxGroups)
    consider(1, std::min(rows_us(a, sh, glu, cus, 16, 2), rows_us(a, sh, glu, cus, 16, 4)));
  return form;
}

// Blocks of 16 in units of four row quads, two items ahead, or of two, three ahead: us (4 / 2),
// 8 of 64 experts, 2048 -> 2 x 1024, 1 / 16 / 64 tokens 6.1 / 21.2 / 29.3, 6.5 / 23.0 / 30.6; 4 of
// 32, 5120 -> 2 x 2176, 1 / 8 / 40 tokens (272 and 544 units on 256 CUs at one) 14.6 / 34.6 / 61.6,
// 13.5 / 33.0 / 62.3; 2 of 8, 8192 -> 1024, 40 tokens 19.7, 24.3. Two workgroups a CU were slower
// throughout (18 to 28 us for 16 tokens).
bool grouped_rows_launch(GroupedArgs& a, bool glu, int cus, int form, hipStream_t s) {
  const int ng = (a.G + kW - 1) / kW;
  if (form > 2 || ng > (form == 2 ? 5 : kMaxGroups)) return false;
  const Shares sh(a);
  const int S = rows_us(a, sh, glu, cus, 16, 4) <= rows_us(a, sh, glu, cus, 16, 2) ? 4 : 2;
  a.P = cus;
  if (glu)
    launch_rows<true>(a, form, S, s);
  else
    launch_rows<false>(a, form, S, s);
  return true;
}

}  // namespace qw4
