// k_grouped_rows: the products grouped by expert where experts have few rows (a decoded
// token, a verify block, a short prompt), for K up to 8 x kMaxGroups groups.
//
// Bound by the chosen experts' weights, each of which a call reads once. The split and
// the sums are k_rows_xr's (rows_xr.hip): blocks of 16 MB rows of an expert against units
// of S row quads of its weight over all of K (gated: a gate unit, then its up unit);
// workgroup p owns a run of units, wave w the groups w, w + 8, ...; the block's
// activations sit in registers while the weights stream through LDS slots, D items
// ahead, across units, blocks and experts; the waves' sums meet in LDS in wave order.
// Weights are used exactly: 128 + q as a bf16 operand, scale and zero point in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>

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

template <bool GLU, int S, int NG, int D, int MB>
__global__ __launch_bounds__(64 * kW) void k_grouped_rows(GroupedArgs a) {
  using L = DmaSlot<4, S>;
  constexpr int kL = L::kLoads;
  constexpr uint32_t kPer = 4 / S;
  constexpr int kArea = 2 * MB * S * 64;   // a wave's sums of a unit, two buffers
  constexpr int kSums = MB == 1 ? 0 : NG * MB * 4;   // MB > 1: a wave's row sums (no registers left)
  // One LDS object: of several the compiler tells the accesses apart and waits for every
  // load into the slots before it reads the sums (vmcnt(0) in place of the counted waits).
  __shared__ u32x4 lds[kW * (D * L::kUnits + kArea + kSums) + (kMaxExperts + 1 + kW + 3) / 4];
  u32x4* const slots = lds;
  f32x4* const red = reinterpret_cast<f32x4*>(slots + kW * D * L::kUnits);
  f32x4* const csum = red + kW * kArea;
  int* const start = reinterpret_cast<int*>(csum + kW * kSums);
  int* const wsum = start + kMaxExperts + 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, q = lane >> 4;
  int all[1];
  expert_starts<64 * kW>(a, start, wsum, all, [](int rows, int) { return (rows + 16 * MB - 1) / (16 * MB); });
  // units of a block (gated: pairs), and this workgroup's run of them
  const int per = (GLU ? a.ld : a.n) / (16 * S);
  const long long total = (long long)all[0] * per;
  const int p = blockIdx.x;
  const long long u0 = p * total / a.P, u1 = (p + 1) * total / a.P;
  int left_units = (int)(u1 - u0);
  if (left_units <= 0) return;
  const int nw = wave < a.G ? (a.G - 1 - wave) / kW + 1 : 0;   // groups of this wave (<= NG)
  constexpr int kPair = GLU ? 2 : 1;
  int left = nw * left_units * kPair;                           // items not yet done

  // a place moves on to the next unit, block and expert
  auto begin = [&](Place& v) __attribute__((always_inline)) {
    v.block = (int)(u0 / per);
    v.unit = (int)(u0 - (long long)v.block * per);
    v.e = expert_of(start, a.E, 1, v.block);
  };
  auto next = [&](Place& v) __attribute__((always_inline)) {
    if (++v.unit == per) {
      v.unit = 0;
      ++v.block;
      while (v.e + 1 < a.E && __builtin_amdgcn_readfirstlane(start[v.e + 1]) <= v.block) ++v.e;
    }
  };

  // The load cursor: unit, its half (gated: gate or up), group; weights of its expert.
  Place lp;
  begin(lp);
  int lhalf = 0, lg = wave, lunits = left_units;
  __amdgpu_buffer_rsrc_t lqw, lsc;
  const uint32_t blocks = (uint32_t)(a.n / kTileN) * (uint32_t)a.G;   // weight blocks of an expert
  auto weights = [&]() __attribute__((always_inline)) {
    const size_t blk = (size_t)lp.e * blocks;
    lqw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(a.qw + blk * kWordsPerBlock), 0,
                                            (int)(blocks * 4096u), 0x00020000);
    lsc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.sc + blk * kMetaU16), 0,
                                            (int)(blocks * (uint32_t)kMetaBytes), 0x00020000);
  };
  weights();
  u32x4* const ring = slots + wave * D * L::kUnits;
  const uint32_t wbase = Fmt<4>::woff(q, c);
  const int up_units = a.epi.up / (16 * S);
  auto load_slot = [&](int j) __attribute__((always_inline)) {
    const bool in = lunits > 0;
    const uint32_t ru = (uint32_t)(lp.unit + lhalf * up_units);
    const uint32_t st0 = ru % kPer * S;
    // past the run: a block past the weights, which loads nothing
    const uint32_t blk = in ? ru / kPer * (uint32_t)a.G + (uint32_t)lg : blocks;
    const uint32_t voff = wbase + st0 * 256u;
    u32x4* const slot = ring + j * L::kUnits;
#pragma unroll
    for (int i = 0; i < S; ++i) dma_load16(lqw, slot + i * 64, voff + i * 256u, blk * 4096u);
    dma_load4(lsc, slot + L::kNQ * 64, lane < 40 ? (uint32_t)lane * 4u : 0u, blk * (uint32_t)kMetaBytes);
    lg += kW;
    if (lg < a.G) return;
    lg = wave;
    if (GLU && lhalf == 0) {
      lhalf = 1;
      return;
    }
    lhalf = 0;
    if (--lunits > 0) {
      const int e = lp.e;
      next(lp);
      if (lp.e != e) weights();
    }
  };
  if (nw > 0) {
#pragma unroll
    for (int j = 0; j < D; ++j) load_slot(j);
  }

  const NibConst k = nib_const();
  const int zsh = 16 * (c & 1);
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
    expert_rows(a, at.e, lo, hi);
    const int nth = __builtin_amdgcn_readfirstlane(at.block - start[at.e]);   // < 0: offsets of no plan
    m0 = __builtin_amdgcn_readfirstlane(lo) + nth * 16 * MB;
    rows = nth < 0 ? 0 : min(__builtin_amdgcn_readfirstlane(hi) - m0, 16 * MB);
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
  float gate[S];   // gated: the gate unit's sums
#pragma unroll
  for (int i = 0; i < S; ++i) gate[i] = 0.f;
  int j = 0, n = 0;   // slot of the next item; units closed
  while (true) {
    const int st0 = (int)((uint32_t)at.unit % kPer) * S;
    for (int half = 0; half < kPair; ++half) {
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
        f32x4 C[MB][S];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < S; ++i) {
            const bf16x8 B = nib8(d.w[i][0][t], k);
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
          for (int i = 0; i < S; ++i) {
            const uint32_t sbits = (d.s[i >> 1] >> (16 * (S == 1 ? (st0 & 1) : (i & 1)))) & 0xffffu;
            const float sf = bf16_bits_to_f32(sbits);
            const float zf = 128.0f + (float)((d.z >> (zsh + 4 * (st0 + i))) & 0xFu);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) acc[mb][i][jj] += sf * (C[mb][i][jj] - zf * cs[jj]);
          }
        }
        // the slot's reads have returned: load the item D ahead into it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (left > D) load_slot(j);
        j = j + 1 == D ? 0 : j + 1;
        --left;
      });
      // Unit sums in wave order; row 4 q + jj by wave jj (mod 4) of one half of the
      // workgroup, the halves taking turns by output unit (MB = 2: a half each row
      // block). Two buffers, one barrier a unit: a buffer is written again two
      // barriers after it was read.
      const int par = n & 1;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < S; ++i) {
          red[wave * kArea + ((par * MB + mb) * S + i) * 64 + lane] = acc[mb][i];
          acc[mb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      lds_barrier<true>();
      if (MB == 2 || (wave >> 2) == ((GLU ? n >> 1 : n) & 1)) {
        const int jj = wave & 3, mb = MB == 2 ? wave >> 2 : 0;
        float v[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const int from = (((par * MB + mb) * S + i) * 64 + lane) * 4 + jj;
          v[i] = reinterpret_cast<const float*>(red)[from];
#pragma unroll
          for (int w = 1; w < kW; ++w) v[i] += reinterpret_cast<const float*>(red + w * kArea)[from];
        }
        if (GLU && half == 0) {
#pragma unroll
          for (int i = 0; i < S; ++i) gate[i] = v[i];
        } else {
          const int m = 16 * mb + 4 * q + jj;
          const int n0 = (int)((uint32_t)at.unit / kPer) * kTileN + 4 * c + st0;
          float f[GLU ? 2 : 1][S];
#pragma unroll
          for (int h = 0; h < (GLU ? 2 : 1); ++h) {
            float b[S];
            load_cols<S>(b, a.epi.bias, (size_t)at.e * a.n + h * a.epi.up + n0);
#pragma unroll
            for (int i = 0; i < S; ++i) f[h][i] = (GLU && h == 0 ? gate[i] : v[i]) + b[i];
          }
          epilogue_act<GLU, S>(f, a.epi.act);
          if (m < rows) {
            uint16_t* y = a.y + (size_t)(m0 + m) * a.ld + n0;
            if constexpr (S == 1) {
              y[0] = to_bf16(f[0][0]);
            } else {
#pragma unroll
              for (int i = 0; i < S / 2; ++i)
                reinterpret_cast<uint32_t*>(y)[i] = pack_bf16x2(f[0][2 * i], f[0][2 * i + 1]);
            }
          }
        }
      }
      ++n;
    }
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

template <bool GLU, int S, int MB>
void launch_ng(const GroupedArgs& a, hipStream_t st) {
  const int ng = (a.G + kW - 1) / kW;
  if (ng <= 3)
    launch<GLU, S, 3, 3, MB>(a, st);
  else if (ng <= 5)
    launch<GLU, S, 5, 3, MB>(a, st);
  else if constexpr (MB == 1)
    launch<GLU, S, kMaxGroups, 3, MB>(a, st);
}

}  // namespace

bool grouped_rows_launch(GroupedArgs& a, bool glu, int cus, hipStream_t s) {
  const int ng = (a.G + kW - 1) / kW;
  const int mean = a.R / a.E;
  if (ng > kMaxGroups || mean > 32) return false;
  const int MB = mean > 12 && ng <= 5 ? 2 : 1;
  const int width = glu ? a.ld : a.n;
  a.P = cus;
  if (glu) {
    MB == 2 ? launch_ng<true, 2, 2>(a, s) : launch_ng<true, 2, 1>(a, s);
  } else {
    MB == 2 ? launch_ng<false, 2, 2>(a, s) : launch_ng<false, 2, 1>(a, s);
  }
  (void)width;
  return true;
}

}  // namespace qw4
