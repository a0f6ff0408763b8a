// Products of activations in 8 bits and INT4 weights (qw4_a8_linear).
//
//   y[m][n] = act(sum_g sx[m][g] sw[n][g] (sum_{k in g} (qw[n][k] - z[n][g]) qx[m][k]) + bias[n]) + res[m][n]
//
// The inner sum is exact in int32 (at most 128 15 127 = 243840) on v_mfma_i32_32x32x32_i8:
// the low nibbles of a packed word less their zero point are four int8 weights, the high
// ones four more, and the activation rows hold their codes in that order. A group's sums
// are scaled into fp32 accumulators.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/qwen_w4a16.h"
#include "a8.h"
#include "epilogue.h"
#include "w4a16_common.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);

namespace {

// ---------------------------------------------------------------------------
// k_a8_tiles: 128 columns (rows of W) x 32 MB rows of x a workgroup of 4 waves; a wave owns
// 32 columns against all the tile's rows, in MB blocks of 32 x 32. Two workgroups fit a CU, so
// that one's vector instructions run beside the other's MFMAs: 4096 rows of 34816 x 5120 take
// 0.88 ms (1.66 POP/s: vector instructions 65% and MFMAs 42% of the cycles), in a first form with one
// workgroup of 8 waves and 256 columns a CU 1.04.
//
// In halves (KS = 2, tiles of up to 4 blocks) a workgroup has 8 waves, the second four take the
// second half of the groups, and the sums meet in LDS: half as many slices for as many waves.
// 77 rows of 5120 x 17408 25 us (28 in whole workgroups), 96 of 34816 x 5120 44 (48), 512 of
// 5120 x 4096 24 (30). Other sizes lose: 256 of 5120 x 17408 47.6 against 46.8.
//
//  * Weights (the MFMA's B operand) come straight into registers, a lane the 32 bytes of
//    its row and half of a group: every weight is unpacked once per workgroup, 7 vector
//    instructions for 8.
//  * Codes (A) go global -> LDS (buffer_load ... lds, whole 128-byte row segments, 1 KiB an
//    instruction), D groups buffered. Row m holds 16-byte chunk c at c ^ g(m), g = (m % 8) ^
//    (m / 8 % 2): the 8 rows that 128 bytes of banks serve, and the 16 of 256 bytes, differ.
//    The scales of the tile's rows lie behind them.
//  * A block's four MFMAs start from M (kA8Magic): its 16 sums a lane are scaled into the
//    accumulators by two instructions each where a conversion, two products and an addition
//    were four: by the lane's weight scale, then by the rows' scales, taken across lanes.
//
// MFMA layout: lane l holds weight row l % 32, inputs of chunks 2 s + l / 32 (s = 0, 1), low
// nibbles and high nibbles an operand each; of the result column l % 32 (a weight row), rows
// (of x) 8 j + 4 (l / 32) + i.
constexpr int kA8Waves = 4;
constexpr int kTileCols = 32 * kA8Waves;
constexpr int kPerCu = 2;   // workgroups; in halves, 1
constexpr int kHalvesMb = 4;   // blocks of a tile in halves at most
constexpr int kA8MostK = 1 << 23;   // 256 rows of codes are offsets of 31 bits

template <int MB>
struct A8Split {
  static constexpr int ACT = 4 * MB / kA8Waves;               // 1 KiB loads of codes a wave and group
  static constexpr int DEPTH = MB <= 2 ? 4 : MB <= 4 ? 3 : 2;   // one or two more: 0 .. 9% slower
  static constexpr int LOADS = ACT + 1 + 4;        // codes, scales, weights (2 + 1 + 1)
  static constexpr int CODES = 32 * MB * 8;        // 16-byte units of a buffer's codes
  static constexpr int UNITS = CODES + kA8Waves * 16;   // and of its scales, 64 a wave's load
  static_assert(4 * MB % kA8Waves == 0 && 32 * MB <= 64 * kA8Waves, "whole loads a wave");
};

struct A8Tiles {
  A8Args a;
  float* slots;              // [P][2] partial tiles
  int tiles_n, tiles_m, map;
  int P, full, U;            // as in the bf16 product: whole tiles [0, full), then U units over P
};

struct A8Weights {
  u32x4 q[2];                // chunks h, 2 + h of the lane's row
  uint32_t s;                // its scale
  uint32_t z;                // zero points of rows r & ~3 .. + 3
};
struct A8Src {               // of a wave's weight tile: blocks and (scale, zero-point) records
  const uint32_t* qw;
  const uint16_t* sc;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t a8_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// Part 0: the words and zero points of group g, part 1: the scale. A group of which there
// is not `some` has a resource of no length: no memory, no branch.
__device__ __forceinline__ void a8_load_weights(A8Weights& w, const A8Src& src, int b, int g, bool some, int lane,
                                                int part) {
  const int r = lane & 31, h = lane >> 5;
  const __amdgpu_buffer_rsrc_t rec = a8_rsrc(src.sc + (size_t)g * kMetaU16, some ? (uint32_t)kMetaBytes : 0u);
  if (part == 0) {
    const __amdgpu_buffer_rsrc_t qw = a8_rsrc(src.qw + (size_t)g * kWordsPerBlock, some ? 4096u : 0u);
    const int pos = tile_pos_of_row(32 * b + r);
#pragma unroll
    for (int s = 0; s < 2; ++s) w.q[s] = __builtin_amdgcn_raw_buffer_load_b128(qw, ((2 * s + h) * 64 + pos) * 16, 0, 0);
    w.z = __builtin_amdgcn_raw_buffer_load_b16(rec, 128 + (8 * b + (r >> 2)) * 2, 0, 0);
  } else {
    w.s = __builtin_amdgcn_raw_buffer_load_b16(rec, (32 * b + r) * 2, 0, 0);
  }
}

// The rows of x that a tile reads.
struct A8Rows {
  const int8_t* q;           // of the tile's first row
  const float* scale;
  uint32_t rows;             // of the tile that there are
};

template <int MB>
__device__ __forceinline__ void a8_load_rows(const A8Args& a, const A8Rows& x, uint32_t voff, u32x4* buf, int g,
                                             bool some, int wave, int lane, int part) {
  using Sp = A8Split<MB>;
  if (part < Sp::ACT) {
    const int rb = part * kA8Waves + wave;   // 8 rows
    const __amdgpu_buffer_rsrc_t rs = a8_rsrc(x.q, some ? x.rows * (uint32_t)a.K : 0u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, buf + rb * 64, 16, voff,
                                             (uint32_t)(8 * rb) * (uint32_t)a.K + (uint32_t)g * kGroup, 0, 0);
  } else {   // 64 scales a wave; those past the tile's rows from a resource of no length
    const __amdgpu_buffer_rsrc_t rs =
        a8_rsrc(x.scale + (size_t)g * a.max_rows, some && wave < (MB + 1) / 2 ? x.rows * 4u : 0u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, buf + Sp::CODES + wave * 16, 4, (uint32_t)(wave * 64 + lane) * 4u, 0, 0, 0);
  }
}

// y[i] += f[i] times lane i's s of each lane's four. One block, whose wait is what a register
// that a vector instruction has written needs before it is read across lanes: whatever the
// compiler puts before it, a copy of s included, is far enough.
__device__ __forceinline__ void a8_fmac_quad(float* y, float s, const float (&f)[4]) {
  asm("s_nop 1\n\t"
      "v_fmac_f32_dpp %0, %4, %5 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %1, %4, %6 quad_perm:[1,1,1,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %2, %4, %7 quad_perm:[2,2,2,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %3, %4, %8 quad_perm:[3,3,3,3] row_mask:0xf bank_mask:0xf"
      : "+&v"(y[0]), "+&v"(y[1]), "+&v"(y[2]), "+&v"(y[3])
      : "v"(s), "v"(f[0]), "v"(f[1]), "v"(f[2]), "v"(f[3]));
}

// One group: the MFMAs over buf with the weights w, while the loads of group gn go out. Behind
// each MFMA the operand that it has taken is read for the block after; a block's sums are
// scaled once its four MFMAs are out, and the fences keep the blocks in order. sx: in each four
// lanes the scales of four neighbouring rows of x, for a v_fmac that takes its factor from one
// of them.
template <int MB>
__device__ __forceinline__ void a8_group(const A8Args& a, float (&acc)[MB][16], const A8Weights& w, A8Weights& wn,
                                         const u32x4* buf, u32x4* nbuf, const A8Rows& x, const A8Src& src, bool more,
                                         uint32_t voff, int b, int gn, int wave, int lane) {
  using Sp = A8Split<MB>;
  const int r = lane & 31, h = lane >> 5;
  const int swz = (r & 7) ^ ((r >> 3) & 1);
  const uint32_t z = ((w.z >> (4 * (r & 3))) & 15u) * 0x01010101u;
  const float* scales = reinterpret_cast<const float*>(buf + Sp::CODES);
  u32x4 v[4];
  auto code = [&](int mb, int o) { return buf[(32 * mb + r) * 8 + ((4 * (o >> 1) + 2 * h + (o & 1)) ^ swz)]; };
#pragma unroll
  for (int o = 0; o < 4; ++o) v[o] = code(0, o);
  float sx[4];               // of rows 8 j + 4 h + lane % 4
  auto row_scales = [&](int mb) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sx[j] = scales[32 * mb + 8 * j + 4 * h + (lane & 3)];
  };
  row_scales(0);
  i32x4 op[4];               // chunk s = 0 low, high nibbles, s = 1 low, high
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      op[2 * s][i] = (int)a8_less(w.q[s][i] & 0x0F0F0F0Fu, z);
      op[2 * s + 1][i] = (int)a8_less((w.q[s][i] >> 4) & 0x0F0F0F0Fu, z);
    }
  const float sw = bf16_bits_to_f32(w.s), less = -kA8Magic * sw;
  i32x16 start;
#pragma unroll
  for (int i = 0; i < 16; ++i) start[i] = kA8Start;
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    i32x16 c = start;
    const float fx[4] = {sx[0], sx[1], sx[2], sx[3]};
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      c = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, v[o]), op[o], c, 0, 0, 0);
      if (mb + 1 < MB) {
        v[o] = code(mb + 1, o);
        if (o == 0) row_scales(mb + 1);
      }
    }
#pragma unroll
    for (int p = 0; p < Sp::ACT + 3; ++p)
      if (p * MB / 2 / (Sp::ACT + 3) == mb) {
        if (p < 2)
          a8_load_weights(wn, src, b, gn, more, lane, p);
        else
          a8_load_rows<MB>(a, x, voff, nbuf, gn, more, wave, lane, p - 2);
      }
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __builtin_fmaf(__int_as_float(c[4 * o + i]), sw, less);
      a8_fmac_quad(acc[mb] + 4 * o, fx[o], f);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int MB, int KS>
__device__ __forceinline__ void a8_segment(const A8Args& a, float (&acc)[MB][16], u32x4* lds, const A8Rows& x,
                                           int tile, int b, int g0, int g1, int half, int wave, int lane) {
  using Sp = A8Split<MB>;
  constexpr int D = Sp::DEPTH;
  const int first = g0;
  const A8Src src{a.qw + (size_t)tile * a.G * kWordsPerBlock, a.sc + (size_t)tile * a.G * kMetaU16};
  // lane i of a load writes slot i % 8 of row i / 8: it fetches the chunk that belongs there
  const uint32_t voff = (uint32_t)(lane >> 3) * (uint32_t)a.K + (uint32_t)((lane & 7) ^ (lane >> 3) ^ (wave & 1)) * 16u;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[mb][i] = 0.f;
  __syncthreads();   // the previous segment's last LDS reads are done
  if (KS == 2) {     // a half of the waves takes a half of the groups
    const int mid = (g0 + g1 + 1) / 2;
    (half ? g0 : g1) = mid;
    lds += half * D * Sp::UNITS;
  }
  const int end = KS == 2 && half ? 2 * g0 - first : g1;   // as many steps for both
  A8Weights w[D];
#pragma unroll
  for (int d = 0; d < D - 1; ++d) {
    const bool in = g0 + d < g1;
#pragma unroll
    for (int p = 0; p <= Sp::ACT; ++p) a8_load_rows<MB>(a, x, voff, lds + d * Sp::UNITS, g0 + d, in, wave, lane, p);
#pragma unroll
    for (int p = 0; p < 2; ++p) a8_load_weights(w[d], src, b, g0 + d, in, lane, p);
  }
  for (int gb = g0; gb < end; gb += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int g = gb + d;
      if (g >= end) break;
      // group g has landed (the D - 2 behind it may be in flight) for every wave, and
      // every wave is done with group g - 1's buffer
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 2) * Sp::LOADS) : "memory");
      if (KS == 2 && g >= g1) break;   // the other half's last
      constexpr int kBack = D - 1;
      a8_group<MB>(a, acc, w[d], w[(d + kBack) % D], lds + d * Sp::UNITS, lds + (d + kBack) % D * Sp::UNITS, x, src,
                   g + kBack < g1, voff, b, g + kBack, wave, lane);
    }
  }
}

__device__ __forceinline__ void a8_tile_coords(const A8Tiles& t, int i, int& tn, int& tm) {
  if (t.map == 2) {   // slices along K: row-major, so an XCD's run shares rows of x
    tm = i / t.tiles_n;
    tn = i - tm * t.tiles_n;
    return;
  }
  const int band = 4 * t.tiles_n;   // bands of 4 row tiles, as in the bf16 product
  const int bd = i / band, w = i % band;
  const int rows = min(4, t.tiles_m - 4 * bd);
  tm = 4 * bd + w % rows;
  tn = w / rows;
}

// Weight tile, half and first output column of wave w in column tile tn. Gated, the second
// half of the waves takes the up rows of the first.
struct A8Wave {
  int tile, b, col;
  bool valid;
};
template <int OUT>
__device__ __forceinline__ A8Wave a8_wave(const A8Args& a, int tn, int w) {
  if (OUT == A8_GLU) {
    constexpr int kHalf = kA8Waves / 2;
    const int t = kHalf / 2 * tn + ((w % kHalf) >> 1);
    const bool ok = t * kTileN < a.ld;
    const int gate = ok ? t : a.ld / kTileN - 1;
    return {gate + (w / kHalf) * (a.epi.up / kTileN), w & 1, t * kTileN + 32 * (w & 1), ok};
  }
  const int t = kA8Waves / 2 * tn + (w >> 1);
  const bool ok = t * kTileN < a.N;
  return {ok ? t : a.N / kTileN - 1, w & 1, t * kTileN + 32 * (w & 1), ok};
}

constexpr uint32_t kA8SlotBytes = 256u * kTileCols * 4;

__device__ __forceinline__ uint32_t a8_slot_off(int vp, int which, int wave, int mb, int lane) {
  return (uint32_t)(vp * 2 + which) * kA8SlotBytes + (uint32_t)((wave * 8 + mb) * 4096 + lane * 16);
}
__device__ __forceinline__ int a8_range_start(const A8Tiles& t, int vp) { return (int)((long long)vp * t.U / t.P); }
__device__ __forceinline__ int a8_owner_of(const A8Tiles& t, int u) { return (int)(((long long)(u + 1) * t.P - 1) / t.U); }

// Tile store: the sums pass through LDS, 32 rows x 128 columns of fp32 a block (16-byte
// chunk c of a row at c ^ (row % 16)), and come back as whole row segments, 8 output
// columns a lane, where gate and up meet, bias and residual are added and the result is
// rounded once.
template <int MB, int OUT, int KS>
__device__ __forceinline__ void a8_store(const A8Args& a, const float (&acc)[MB][16], u32x4* lds, int m0, int tn,
                                         int half, int wave, int lane) {
  constexpr bool GLU = OUT == A8_GLU;
  constexpr int kFits = KS * A8Split<MB>::DEPTH * A8Split<MB>::UNITS / (8 * kTileCols);
  constexpr int kPass = kFits < MB ? kFits : MB;   // blocks of 16 KiB at a time
  static_assert(kPass >= 1, "a block fits the buffers");
  constexpr int kCols = GLU ? kTileCols / 2 : kTileCols, kChunks = kTileCols / 4, kLanes = kCols / 8, kRows = 64 * kA8Waves * KS / kLanes;
  const int r = lane & 31, h = lane >> 5;
  const int t = (KS == 2 ? half * kA8Waves + wave : wave) * 64 + lane, cl = t % kLanes, rl = t / kLanes;
  const int col = tn * kCols + 8 * cl;
  const bool in = col < a.ld;
  float bias[GLU ? 2 : 1][8];
  if (OUT != A8_F32 && in) load_bias<GLU>(bias, a.epi, col);
#pragma unroll
  for (int p0 = 0; p0 < MB; p0 += kPass) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPass; ++k) {
      if (p0 + k >= MB || (KS == 2 && half)) break;
      const float(&v)[16] = acc[p0 + k < MB ? p0 + k : 0];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = 8 * (i >> 2) + 4 * h + (i & 3);
        reinterpret_cast<float*>(lds + (32 * k + row) * kChunks + ((8 * wave + (r >> 2)) ^ (row & 15)))[r & 3] = v[i];
      }
    }
    __syncthreads();
    const int rows = 32 * (p0 + kPass <= MB ? kPass : MB - p0);
    for (int row = rl; row < rows; row += kRows) {
      const int m = m0 + 32 * p0 + row;
      if (!in || m >= a.M) continue;
      const size_t at = (size_t)m * a.ld + col;
      if constexpr (OUT == A8_F32) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<u32x4*>(static_cast<float*>(a.y) + at + 4 * c) = lds[row * kChunks + ((2 * cl + c) ^ (row & 15))];
      } else {
        u32x4 res = {0u, 0u, 0u, 0u};
        if (a.epi.res) res = *reinterpret_cast<const u32x4*>(a.epi.res + at);
        float v[GLU ? 2 : 1][8];
#pragma unroll
        for (int j = 0; j < (GLU ? 2 : 1); ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const u32x4 w = lds[row * kChunks + ((kChunks / 2 * j + 2 * cl + c) ^ (row & 15))];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][4 * c + i] = __uint_as_float(w[i]) + bias[j][4 * c + i];
          }
        epilogue_act<GLU>(v, a.epi.act);
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + at) = add_round8(v[0], res);
      }
    }
  }
}

// The second half's sums to the first's.
template <int MB>
__device__ __forceinline__ void a8_join(float (&acc)[MB][16], u32x4* lds, int half, int wave, int lane) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u32x4& at = lds[((wave * MB + mb) * 4 + k) * 64 + lane];
      if (half)
        at = u32x4{__float_as_uint(acc[mb][4 * k]), __float_as_uint(acc[mb][4 * k + 1]),
                   __float_as_uint(acc[mb][4 * k + 2]), __float_as_uint(acc[mb][4 * k + 3])};
    }
  __syncthreads();
  if (half) return;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const u32x4 v = lds[((wave * MB + mb) * 4 + k) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[mb][4 * k + i] += __uint_as_float(v[i]);
    }
}

template <int MB, int OUT, int KS>
__global__ __launch_bounds__(64 * kA8Waves * KS, 2) void k_a8_tiles(A8Tiles t) {
  using Sp = A8Split<MB>;
  __shared__ u32x4 lds[KS * Sp::DEPTH * Sp::UNITS];
  static_assert(KS == 1 || 1024 * MB <= KS * Sp::DEPTH * Sp::UNITS, "the join's sums fit the buffers");
  const A8Args& a = t.a;
  const int waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wave = KS == 2 ? waves % kA8Waves : waves, half = KS == 2 ? waves / kA8Waves : 0;
  float acc[MB][16];
  int vp = blockIdx.x;
  if (t.map) vp = (vp & 7) * (t.P >> 3) + (vp >> 3);   // each XCD a contiguous run (P % 8 == 0)
  if (t.map == 2) {   // the runs go over slices, then tiles
    const int nt = t.tiles_n * t.tiles_m, sl = vp / nt;
    vp = (vp - sl * nt) * (t.P / nt) + sl;
  }
  const int u1 = a8_range_start(t, vp + 1);
  int u = a8_range_start(t, vp), i = vp, which = 0;
  for (;;) {   // whole tiles, then the units of this workgroup's range
    int tile = i, g0 = 0, g1 = a.G;
    if (i < t.full) {
      i += t.P;
    } else if (u < u1) {
      const int ts = u / a.G;
      g0 = u - ts * a.G;
      g1 = min(a.G, u1 - ts * a.G);
      tile = t.full + ts;
      u = ts * a.G + g1;
    } else {
      break;
    }
    int tn, tm;
    a8_tile_coords(t, tile, tn, tm);
    const int m0 = tm * 32 * MB;
    const A8Wave w = a8_wave<OUT>(a, tn, wave);
    const A8Rows x{a.q + (size_t)m0 * a.K, a.scale + m0, (uint32_t)min(a.M - m0, 32 * MB)};
    a8_segment<MB, KS>(a, acc, lds, x, w.tile, w.b, g0, g1, half, wave, lane);
    if constexpr (KS == 2) a8_join<MB>(acc, lds, half, wave, lane);
    if (g0 == 0 && g1 == a.G) {
      a8_store<MB, OUT, KS>(a, acc, lds, m0, tn, half, wave, lane);
    } else if (half == 0) {   // the range's first tile to the first slot, its last to the second
      const __amdgpu_buffer_rsrc_t rs = a8_rsrc(t.slots, 2u * t.P * kA8SlotBytes);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          __builtin_amdgcn_raw_buffer_store_b128(
              u32x4{__float_as_uint(acc[mb][4 * k]), __float_as_uint(acc[mb][4 * k + 1]),
                    __float_as_uint(acc[mb][4 * k + 2]), __float_as_uint(acc[mb][4 * k + 3])},
              rs, a8_slot_off(vp, which, wave, mb, lane) + 1024 * k, 0, 0);
    }
    if (tile >= t.full) which = 1;
  }
}

// The cut tiles: a wave sums a quarter of a block (wave w, m-block mb, rows 8 j .. 8 j + 7 of
// it; gated: of gate and up) over its pieces, in order, kAhead of them loaded at a time, and
// stores it: a lane has four rows of a column, and takes four columns of a row from its four.
constexpr int kA8Quarters = 4;

// A 4 x 4 block in four lanes, turned: v[i] of lane j to v[j] of lane i.
template <int CTRL>
__device__ __forceinline__ void a8_swap(float& low, float& high, bool second) {
  const int give = __float_as_int(second ? low : high);
  const float got = __int_as_float(__builtin_amdgcn_update_dpp(give, give, CTRL, 0xf, 0xf, false));
  low = second ? got : low;
  high = second ? high : got;
}
__device__ __forceinline__ void a8_turn_quad(float (&v)[4], int lane) {
  const bool odd = lane & 1, upper = lane & 2;
  a8_swap<0xB1>(v[0], v[1], odd);     // quad_perm [1, 0, 3, 2]
  a8_swap<0xB1>(v[2], v[3], odd);
  a8_swap<0x4E>(v[0], v[2], upper);   // quad_perm [2, 3, 0, 1]
  a8_swap<0x4E>(v[1], v[3], upper);
}

template <int MB, int OUT>
__global__ __launch_bounds__(64) void k_a8_fixup(A8Tiles t) {
  constexpr bool GLU = OUT == A8_GLU;
  constexpr int kPer = (GLU ? kA8Waves / 2 : kA8Waves) * MB * kA8Quarters, NP = GLU ? 2 : 1, kAhead = 12;
  const A8Args& a = t.a;
  const int ts = blockIdx.x / kPer, part = blockIdx.x % kPer;
  const int j = part % kA8Quarters, mb = part / kA8Quarters % MB, w = part / (kA8Quarters * MB);
  const int p0 = a8_owner_of(t, ts * a.G), p1 = a8_owner_of(t, ts * a.G + a.G - 1);
  if (p0 == p1) return;   // stored whole
  int tn, tm;
  a8_tile_coords(t, t.full + ts, tn, tm);
  const A8Wave wv = a8_wave<OUT>(a, tn, w);
  const int lane = threadIdx.x, m0 = tm * 32 * MB + 32 * mb + 8 * j, m = m0 + 4 * (lane >> 5) + (lane & 3);
  if (!wv.valid || m0 >= a.M) return;
  const __amdgpu_buffer_rsrc_t rs = a8_rsrc(t.slots, 2u * t.P * kA8SlotBytes);
  float acc[NP][4] = {};
  for (int pp = p0; pp <= p1; pp += kAhead) {
    u32x4 v[kAhead][NP];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int q = pp + k;
      const bool live = q <= p1;   // others read out of range: zeros, without memory
      const int which = live && a8_range_start(t, q) / a.G == ts ? 0 : 1;
#pragma unroll
      for (int p = 0; p < NP; ++p)
        v[k][p] = __builtin_amdgcn_raw_buffer_load_b128(
            rs, live ? a8_slot_off(q, which, w + kA8Waves / 2 * p, mb, lane) + 1024 * j : 0xfffffff0u, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[p][i] += __uint_as_float(v[k][p][i]);
  }
#pragma unroll
  for (int p = 0; p < NP; ++p) a8_turn_quad(acc[p], lane);
  if (m >= a.M) return;
  const int col = wv.col + (lane & 28);
  const size_t at = (size_t)m * a.ld + col;
  if constexpr (OUT == A8_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) = f32x4{acc[0][0], acc[0][1], acc[0][2], acc[0][3]};
  } else {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      u32x2 bv = {0u, 0u};
      if (a.epi.bias) bv = *reinterpret_cast<const u32x2*>(a.epi.bias + p * a.epi.up + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[p][i] += bf16_bits_to_f32((bv[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
    epilogue_act<GLU>(acc, a.epi.act);
    u32x2 q = {0u, 0u};
    if (a.epi.res) q = *reinterpret_cast<const u32x2*>(a.epi.res + at);
    const float* f = acc[0];
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + at) =
        u32x2{pack_bf16x2(f[0] + bf16_bits_to_f32(q[0] & 0xffffu), f[1] + bf16_bits_to_f32(q[0] >> 16)),
              pack_bf16x2(f[2] + bf16_bits_to_f32(q[1] & 0xffffu), f[3] + bf16_bits_to_f32(q[1] >> 16))};
  }
}

// How a call is cut: ks 1 or, in halves, 2; tiles of 32 mb rows; schedule 0 whole tiles, 2
// whole rounds and the rest's units spread over all workgroups, 3 every tile in S slices;
// estimated us.
struct A8Plan {
  int ks, mb, tiles_n, tiles_m, pick, S;
  double cost;
};

// The best cut of tiles of mb rows. The estimate's figures are fitted to 2100 timed calls on
// MI355X (15 projections from 2048x2048 to 248320x5120, 24 to 4096 rows, every ks, mb,
// schedule and S, with steps some 4% longer than now): over its 110 sizes the pick is 1.2% (geometric mean) from the fastest of
// all, 11% at worst (64 rows and fewer of 2048x2048). A (tile, group) step takes `one` us with
// one workgroup on a CU and `two` with two, or with one in halves; then come storing a tile, the
// second kernel that joins slices, and their partial tiles' traffic. All units over all
// workgroups (ranges that begin and end anywhere) was the fastest by 0.3% in the mean and is
// not kept.
A8Plan a8_plan(int M, int cols, int G, int ks, int mb, int cus, bool ws_ok) {
  A8Plan p{ks, mb, (cols + kTileCols - 1) / kTileCols, (M + 32 * mb - 1) / (32 * mb), 0, 1, 0.};
  const int at_once = ks == 2 ? 1 : kPerCu, half = (G + ks - 1) / ks;
  const long long nt = (long long)p.tiles_n * p.tiles_m, most = at_once * cus, rem = nt % most;
  const double one = 0.23 + 0.21 * mb, two = ks == 2 ? 0.57 + 0.27 * mb : 0.54 + 0.23 * mb;
  const double store = (ks == 2 ? 0.08 : 0.86) * mb;
  auto whole = [&](long long tiles) {   // of the CU with most tiles, as many at once as it holds
    const long long n = (tiles + cus - 1) / cus;
    return (double)(n / at_once) * (half * two + store) + (double)(n % at_once) * (half * one + store);
  };
  p.cost = whole(nt);
  if (!ws_ok || nt * G >= (1LL << 31)) return p;
  auto take = [&](int pick, int S, double c) {
    if (c < p.cost) {
      p.pick = pick;
      p.S = S;
      p.cost = c;
    }
  };
  if (nt > most && rem && rem * G >= most)
    take(2, 1, whole(nt - rem) + (double)rem * half / most * two + 3.1 + 4.45 * mb);
  for (int S = 2; S <= 64 && nt * S <= most && 2 * S <= G; ++S) {
    const long long P = nt * S;
    if (P % 8) continue;   // runs of workgroups on each XCD
    const int steps = ((G + S - 1) / S + ks - 1) / ks;
    take(3, S, steps * (P <= cus && ks == 1 ? one : two) + 3.9 + 4.71 * (double)P / (kPerCu * cus) * mb);
  }
  return p;
}

template <int OUT, int MB>
void launch_tiles(const A8Tiles& t, int ks, int grid, int nt, hipStream_t s) {
  if (ks == 1) {
    k_a8_tiles<MB, OUT, 1><<<grid, 64 * kA8Waves, 0, s>>>(t);
  } else if constexpr (MB <= kHalvesMb) {
    k_a8_tiles<MB, OUT, 2><<<grid, 128 * kA8Waves, 0, s>>>(t);
  }
  if (t.full != nt)
    k_a8_fixup<MB, OUT>
        <<<(nt - t.full) * (OUT == A8_GLU ? kA8Waves / 2 : kA8Waves) * MB * kA8Quarters, 64, 0, s>>>(t);
}

template <int OUT>
int run(const A8Args& a, qw4_workspace* ws, hipStream_t s) {
  const int cus = device_cus(), cols = OUT == A8_GLU ? 2 * a.ld : a.ld;
  if (a8_few(OUT, a, cus, s)) {
    QW4_LAUNCH_CHECK();
    return QW4_OK;
  }
  const bool ws_ok = ws && ws->buf && ((uintptr_t)ws->buf & 255) == 0 && cus % 8 == 0 &&
                     ws->bytes >= 2ull * kPerCu * cus * kA8SlotBytes;
  A8Plan p = a8_plan(a.M, cols, a.G, 1, 8, cus, ws_ok);
  for (int ks = 1; ks <= 2; ++ks)
    for (int mb = ks == 2 ? kHalvesMb : 6; mb >= 1; --mb) {
      const A8Plan q = a8_plan(a.M, cols, a.G, ks, mb, cus, ws_ok);
      if (q.cost < p.cost) p = q;
    }
  const long long tiles = (long long)p.tiles_n * p.tiles_m;
  if (tiles > 0x7fffffffLL / 64) return QW4_ERR_SHAPE;
  const int nt = (int)tiles;
  A8Tiles t{a, nullptr, p.tiles_n, p.tiles_m, nt % 8 == 0, nt, nt, 0};
  int grid = nt;
  if (p.pick) {
    t.slots = static_cast<float*>(ws->buf);
    const int most = (p.ks == 2 ? 1 : kPerCu) * cus;
    t.P = grid = p.pick == 3 ? nt * p.S : most;
    t.full = p.pick == 2 ? nt - nt % most : 0;
    t.U = (nt - t.full) * a.G;
    t.map = p.pick == 3 ? 2 : 1;
  }
  switch (p.mb) {
    case 1: launch_tiles<OUT, 1>(t, p.ks, grid, nt, s); break;
    case 2: launch_tiles<OUT, 2>(t, p.ks, grid, nt, s); break;
    case 3: launch_tiles<OUT, 3>(t, p.ks, grid, nt, s); break;
    case 4: launch_tiles<OUT, 4>(t, p.ks, grid, nt, s); break;
    case 5: launch_tiles<OUT, 5>(t, p.ks, grid, nt, s); break;
    case 6: launch_tiles<OUT, 6>(t, p.ks, grid, nt, s); break;
    default: launch_tiles<OUT, 8>(t, p.ks, grid, nt, s);
  }
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

int check_call(const void* y, const qw4_weights* w, const qw4_a8* a, int T) {
  int st = check_weights_public(w);
  if (st) return st;
  if (!y) return QW4_ERR_NULL;
  if (T < 1) return QW4_ERR_M;
  st = check_a8(a, 0, T);
  if (st) return st;
  if (a->in_f != w->in_f || a->in_f > kA8MostK) return QW4_ERR_SHAPE;
  if ((uintptr_t)y & 15) return QW4_ERR_ALIGN;
  return QW4_OK;
}

A8Args args_of(void* y, const qw4_weights* w, const qw4_a8* a, int T, const Epilogue& e) {
  return {w->qweight, w->scale, a->q, a->scale, y, T, w->out_f, w->in_f, w->num_groups,
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
  const A8Args g = args_of(y, w, a, T, Epilogue{bias, residual, act, glu ? w->out_f / 2 : 0});
  return glu ? run<A8_GLU>(g, ws, (hipStream_t)stream) : run<A8_EPI>(g, ws, (hipStream_t)stream);
}

int qw4_a8_linear_f32(float* y, const qw4_weights* w, const qw4_a8* a, int T, qw4_workspace* ws, void* stream) {
  const int st = check_call(y, w, a, T);
  if (st) return st;
  return run<A8_F32>(args_of(y, w, a, T, Epilogue{}), ws, (hipStream_t)stream);
}

}  // extern "C"
