// Prefill W4A16 GEMM: C [M][N] = A [M][K] @ W^T, bf16 in/out, fp32 accumulate.
//
// The reference dequantizes whole weight tiles to a bf16 workspace and calls
// cublasGemmEx (src/kernels/gemm_w4a16.cu:63-88). Here the dequant is fused
// into one gfx950 kernel: each wave converts its packed weight rows in
// registers to exactly RNE((q - z) * s) -- the reference's k_dequant_rows
// arithmetic (gemm_w4a16.cu:26-36) -- and feeds them to bf16 MFMA against
// activation tiles staged in LDS. Tiles that would leave CUs idle in a last
// partial round are instead split across workgroups (stream-K, hybrid or
// split-K) when a workspace is given; the workspace then holds fp32 partial
// tiles, summed in a fixed order by a second kernel.
#include <hip/hip_runtime.h>

#include <atomic>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "../../include/qwen_w4a16.h"
#include "gemm_tile.h"
#include "w4a16_common.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);

namespace {

// Outputs of k_gemm: the product in bf16; with an epilogue; with an epilogue that
// joins gate and up (C, residual and ld of half the weight's rows), the operands in
// bf16 or, with a workspace for them, in fp16.
enum { GEMM_PLAIN = 0, GEMM_EPI = 1, GEMM_GLU = 2, GEMM_GLU16 = 3 };
constexpr bool gemm_glu(int out) { return out == GEMM_GLU || out == GEMM_GLU16; }

struct GemmArgs {
  const uint32_t* qw;
  const uint16_t* sc;
  const uint16_t* zr;
  const uint16_t* A;
  uint16_t* C;
  float* slots;         // stream-K: [P][2] fp32 partial tiles
  int M, N, K, G, tiles_n, tiles_m, map;
  int bm;               // rows of a tile (8-wave variants; 32 MB in the default kernels)
  int P;                // workgroups
  // map: 0 blockIdx order; 1 XCD-contiguous runs of workgroups; 2 split-K:
  // XCD-contiguous runs over (k-slice, tile row-major), P / tiles slices
  int full;             // tiles [0, full) are done whole, P at a time
  int U;                // (tile, group) units of tiles [full, tiles), split over P
  Epilogue epi;
  int ld;               // row stride of C and the residual
  const int *rexp, *cexp;   // GEMM_GLU16: exponents of rows and columns
};

// Linear tile index -> (tn, tm), in bands of 4 M-tiles: consecutive tiles
// share an activation tile (and, 4 apart, a weight tile), so the ~32
// workgroups an XCD runs at once touch ~4 activation and ~8 weight tiles.
__device__ __forceinline__ void g2_tile_coords(const GemmArgs& a, int t, int& tn, int& tm) {
  if (a.map == 2) {   // split-K: row-major, so an XCD's run shares the rows of A
    tm = t / a.tiles_n;
    tn = t - tm * a.tiles_n;
    return;
  }
  const int band = 4 * a.tiles_n;
  const int b = t / band, w = t % band;
  const int rows = min(4, a.tiles_m - 4 * b);
  tm = 4 * b + w % rows;
  tn = w / rows;
}

// What a wave of column tile tn computes: weight tile and first half, and the first
// column of its output. Gated: a workgroup's 128 output columns are two gate tiles and
// the up tiles `up` rows on; a wave takes one half of a gate tile and the same half of
// its up tile, so that gate and up of a column meet in one lane.
struct WaveTile {
  int tile, b0, col;
  bool valid;
};
template <int OUT>
__device__ __forceinline__ WaveTile g2_wave_tile(const GemmArgs& a, int tn, int wt, int b0) {
  if (gemm_glu(OUT)) {
    const int t = tn * 2 + (wt >> 1);
    return {t, wt & 1, t * kTileN + 32 * (wt & 1), t * kTileN < a.ld};
  }
  const int t = tn * 4 + wt;
  return {t, b0, t * kTileN + 32 * b0, t * kTileN < a.N};
}

// Rows of a tile. The 8-wave variants exist for MB = 8 only and run the plan's
// lower tiles in it (rows past bm read as zeros and are not stored), so that a
// call is cut the same way under every variant.
template <int NW, int MB>
__device__ __forceinline__ int g2_tile_rows(const GemmArgs& a) {
  return NW == 8 ? a.bm : 32 * MB;
}
// First row past the tile at m0 that is not stored.
template <int NW>
__device__ __forceinline__ int g2_row_end(const GemmArgs& a, int m0) {
  return NW == 8 ? min(a.M, m0 + a.bm) : a.M;
}

// Tile store. Accumulator layout: lane holds column m = 32 mb + r and rows
// 8 jq + 4 h + i, i.e. output columns n = 64 tile + 4 (8 b + 2 jq + h) + i.
// Stored from that layout directly, a store instruction writes 8 bytes per
// lane to 32 rows (16-byte pieces of 32 lines), and the partial-line requests
// bound the store of a tile (gate M = 4096: ~10% of the kernel's time). So the
// tile goes through LDS and every store instruction writes whole 128-byte row
// segments of C: each wave stages its own region of the 128 KiB activation
// buffers (its rows x NH * 64 bytes, 16-byte chunk c of row m at c ^ (m %
// CPR)) -- after a wait and a barrier, so that all waves are done with the
// segment's operand reads and their loads have landed -- and reads it back
// row by row. Measured: gate M = 4096 0.617 -> 0.601 ms.
template <int NH, int NW, int MB>
__device__ __forceinline__ void g2_store_staged(const GemmArgs& a,
                                                const f32x16v (&acc)[NH][G2Split<NH, NW, MB>::MBW],
                                                u32x4* lds, int m0, int tile, int b0, int mw,
                                                bool valid, int wave, int lane) {
  constexpr int MBW = G2Split<NH, NW, MB>::MBW;
  constexpr int CPR = NH * 4;                      // 16-byte chunks per staged row
  constexpr int ROWS = MBW * 32;
  constexpr int RPI = 64 / CPR;                    // rows per read-back instruction
  const int r = lane & 31, h = lane >> 5;
  g2_wait_vm0();
  __syncthreads();
  u32x4* reg = lds + wave * (ROWS * CPR);
  uint32_t* reg32 = reinterpret_cast<uint32_t*>(reg);
#pragma unroll
  for (int mb = 0; mb < MBW; ++mb) {
    const int row = 32 * mb + r;
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq) {
        const int c = (4 * j + jq) ^ (row % CPR);
        const u32x2 o = {pack_bf16x2(acc[j][mb][4 * jq], acc[j][mb][4 * jq + 1]),
                         pack_bf16x2(acc[j][mb][4 * jq + 2], acc[j][mb][4 * jq + 3])};
        *reinterpret_cast<u32x2*>(reg32 + (row * CPR + c) * 4 + 2 * h) = o;
      }
  }
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
  if (!valid) return;
  const int cl = lane % CPR;
#pragma unroll
  for (int t = 0; t < ROWS / RPI; ++t) {
    const int row = RPI * t + lane / CPR;
    const u32x4 v = reg[row * CPR + (cl ^ (row % CPR))];
    const int m = m0 + 32 * mw + row;
    if (m < g2_row_end<NW>(a, m0))
      *reinterpret_cast<u32x4*>(a.C + (size_t)m * a.N + tile * kTileN + 32 * b0 + 8 * cl) = v;
  }
}

// Stream-K partial tiles. Each workgroup has two fp32 slots (for its first
// and its last tile), laid out [wave][pair][i][lane]: 16-byte piece i of a
// lane's 64 bytes at 1024 i + 16 lane, so that every store (and the fixup's
// every load) covers 1 KiB contiguously; lane-major 64-byte runs made each
// instruction write 16-byte pieces of 32 lines (down M = 512: 0.111 -> 0.098
// ms). A workgroup whose range cuts a tile writes its partial there; a second
// kernel (k_gemm_fixup, stream-ordered after this one) sums each cut tile's
// slots in workgroup order -- a fixed order, so results are bitwise
// reproducible -- and stores the tile.
constexpr uint32_t kSlotBytes = (uint32_t)G2_BM * G2_BN * 4;   // 256 KiB

// idx: the wave's (half, m-block) pair j * MBW + mb, of `units` per wave.
__device__ __forceinline__ uint32_t g2_slot_off(int vp, int which, int wave, int units, int idx,
                                                int lane) {
  return (uint32_t)(vp * 2 + which) * kSlotBytes + (uint32_t)((wave * units + idx) * 4096 + lane * 16);
}

template <int NH, int NW, int MB>
__device__ __forceinline__ void g2_slot_store(__amdgpu_buffer_rsrc_t rs,
                                              const f32x16v (&acc)[NH][G2Split<NH, NW, MB>::MBW],
                                              int vp, int which, int wave, int lane) {
  constexpr int MBW = G2Split<NH, NW, MB>::MBW;
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int mb = 0; mb < MBW; ++mb) {
      const uint32_t off = g2_slot_off(vp, which, wave, NH * MBW, j * MBW + mb, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 v = {__float_as_uint(acc[j][mb][4 * i]), __float_as_uint(acc[j][mb][4 * i + 1]),
                         __float_as_uint(acc[j][mb][4 * i + 2]),
                         __float_as_uint(acc[j][mb][4 * i + 3])};
        __builtin_amdgcn_raw_buffer_store_b128(v, rs, off + 1024 * i, 0, 0);
      }
    }
}

// Ranges over the split tiles' units (unit u: tile full + u / G).
__device__ __forceinline__ int g2_range_start(const GemmArgs& a, int vp) {
  return (int)((long long)vp * a.U / a.P);
}
// Largest vp with g2_range_start(vp) <= u.
__device__ __forceinline__ int g2_owner_of(const GemmArgs& a, int u) {
  return (int)(((long long)(u + 1) * a.P - 1) / a.U);
}

// The cut tiles' fp32 partials are summed by many small blocks: block
// (tile ts, main-kernel wave w, part) owns the pairs [part * 2, part * 2 + 2)
// of wave w's region (the slot layout [wave][pair][i][lane] keeps them
// contiguous), so a cut tile is read by 32 blocks at once instead of one
// workgroup (one workgroup summing its tile inside k_gemm measured slower). A block loads kFixAhead pieces before it adds them, in piece
// order, so that the loads of a tile split many ways overlap instead of
// paying one memory latency per piece. Tiles a single workgroup covered were
// stored by the main kernel.
constexpr int kFixAhead = 4;

//
// In a gated product a block owns the two pairs of one m-block: gate and up.
template <int NH, int NW, int MB, int OUT>
__global__ __launch_bounds__(64) void k_gemm_fixup(GemmArgs a) {
  using Sp = G2Split<NH, NW, MB>;
  constexpr int MBW = Sp::MBW;
  constexpr int kPer = 2;   // (half, m-block) pairs per block
  constexpr int kFixBlocksPerTile = NW * Sp::FIXP;
  static_assert(Sp::UNITS % kPer == 0, "whole pairs per block");
  const int ts = blockIdx.x / kFixBlocksPerTile;   // split tile full + ts
  const int wave = (blockIdx.x / Sp::FIXP) % NW;
  const int part = blockIdx.x % Sp::FIXP;
  const int t = a.full + ts;
  const int p0 = g2_owner_of(a, ts * a.G), p1 = g2_owner_of(a, ts * a.G + a.G - 1);
  if (p0 == p1) return;
  const int lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  int wt, b0, mw;
  Sp::coords(wave, wt, b0, mw);
  int tn, tm;
  g2_tile_coords(a, t, tn, tm);
  const WaveTile w = g2_wave_tile<OUT>(a, tn, wt, b0);
  if (!w.valid) return;
  auto pair = [&](int e) { return gemm_glu(OUT) ? e * MBW + part : part * kPer + e; };
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(a.slots, 0, (int)(2u * a.P * kSlotBytes), 0x00020000);
  f32x16v acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = f32x16v{};
  for (int pp = p0; pp <= p1; pp += kFixAhead) {
    u32x4 v[kFixAhead][kPer][4];
#pragma unroll
    for (int k = 0; k < kFixAhead; ++k) {
      // pieces past p1 read out of range (zeros, no memory access) and are
      // never added: adding +0 would turn a -0 sum into +0
      const int q = pp + k;
      const bool live = q <= p1;
      const int which = (live && g2_range_start(a, q) / a.G == ts) ? 0 : 1;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t off =
            live ? g2_slot_off(q, which, wave, Sp::UNITS, pair(e), lane) : 0x80000000u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[k][e][i] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 1024 * i, 0, 0);
      }
    }
#pragma unroll
    for (int k = 0; k < kFixAhead; ++k) {
      if (pp + k > p1) break;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[e][4 * i + c] += __uint_as_float(v[k][e][i][c]);
    }
  }
  // pair index j * MBW + mb (g2_slot_store's order)
  const int m0 = tm * g2_tile_rows<NW, MB>(a);
  if constexpr (OUT != GEMM_PLAIN) {
    // straight from the accumulators' layout: 4 columns of a row at a time
    constexpr int kOuts = gemm_glu(OUT) ? 1 : kPer;
#pragma unroll
    for (int e = 0; e < kOuts; ++e) {
      const int idx = pair(e), mb = idx % MBW;
      const int m = m0 + 32 * (mw + mb) + r;
      const bool in = m < g2_row_end<NW>(a, m0);
      const int col = w.col + (gemm_glu(OUT) ? 0 : 32 * (idx / MBW)) + 4 * h;
      float v[gemm_glu(OUT) ? 2 : 1][16];
#pragma unroll
      for (int j = 0; j < (gemm_glu(OUT) ? 2 : 1); ++j)
#pragma unroll
        for (int jq = 0; jq < 4; ++jq) {
          u32x2 b = {0u, 0u};
          if (a.epi.bias) b = *reinterpret_cast<const u32x2*>(a.epi.bias + j * a.epi.up + col + 8 * jq);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f = acc[e + j][4 * jq + i];
            if (OUT == GEMM_GLU16 && in)
              f = __builtin_ldexpf(f, a.rexp[m] + a.cexp[j * a.epi.up + col + 8 * jq + i]);
            v[j][4 * jq + i] = f + bf16_bits_to_f32((b[i >> 1] >> (16 * (i & 1))) & 0xffffu);
          }
        }
      epilogue_act<gemm_glu(OUT)>(v, a.epi.act);
      if (!in) continue;
#pragma unroll
      for (int jq = 0; jq < 4; ++jq) {
        const size_t at = (size_t)m * a.ld + col + 8 * jq;
        u32x2 q = {0u, 0u};
        if (a.epi.res) q = *reinterpret_cast<const u32x2*>(a.epi.res + at);
        const float* f = &v[0][4 * jq];
        *reinterpret_cast<u32x2*>(a.C + at) =
            u32x2{pack_bf16x2(f[0] + bf16_bits_to_f32(q[0] & 0xffffu), f[1] + bf16_bits_to_f32(q[0] >> 16)),
                  pack_bf16x2(f[2] + bf16_bits_to_f32(q[1] & 0xffffu), f[3] + bf16_bits_to_f32(q[1] >> 16))};
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int idx = part * kPer + e, j = idx / MBW, mb = idx % MBW;
    const int m = m0 + 32 * (mw + mb) + r;
    if (m >= g2_row_end<NW>(a, m0)) continue;
    uint16_t* crow = a.C + (size_t)m * a.N + w.tile * kTileN;
#pragma unroll
    for (int jq = 0; jq < 4; ++jq) {
      const u32x2 o = {pack_bf16x2(acc[e][4 * jq], acc[e][4 * jq + 1]),
                       pack_bf16x2(acc[e][4 * jq + 2], acc[e][4 * jq + 3])};
      *reinterpret_cast<u32x2*>(crow + 4 * (8 * (b0 + j) + 2 * jq + h)) = o;
    }
  }
}

template <int NH, int NW, int MB, int OUT>
__global__ __launch_bounds__(64 * NW, 1) void k_gemm(GemmArgs a) {
  static_assert(OUT == GEMM_PLAIN || (NH == 2 && NW == 4), "epilogues: the default kernel");
  using Sp = G2Split<NH, NW, MB>;
  constexpr int MBW = Sp::MBW;              // m-blocks per wave
  const int bm = g2_tile_rows<NW, MB>(a);   // rows of a tile
  __shared__ u32x4 lds[Sp::DEPTH][32 * MB * 16];   // [row][16 swizzled chunks]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // wave-uniform
  const int lane = threadIdx.x & 63;
  int wt, b0, mw;
  Sp::coords(wave, wt, b0, mw);
  f32x16v acc[NH][MBW];

  // Virtual workgroup vp (XCD x owns a contiguous run of vp) first does the
  // whole tiles vp, vp + P, ... < full, then the units [start(vp),
  // start(vp + 1)) of the U = (tiles - full) x G units of the remaining
  // tiles: ranges that cut a tile (stream-K) are combined through slots.
  // P = tiles, full = tiles: one whole tile per workgroup.
  int vp = a.map ? g2_xcd_order(blockIdx.x, a.P) : (int)blockIdx.x;
  if (a.map == 2) {
    // Split-K: the P = tiles x S ranges are the S k-slices of each tile (vp =
    // tile S + slice). The XCD runs go over slices, then tiles row-major, so
    // the ~30 workgroups of an XCD work on the same k-slice of one or two
    // rows of tiles: they share A's rows in their L2, at the same k.
    const int nt = a.tiles_n * a.tiles_m, S = a.P / nt;
    const int sl = vp / nt, ts = vp - sl * nt;
    vp = ts * S + sl;
  }
  const int u0 = g2_range_start(a, vp), u1 = g2_range_start(a, vp + 1);
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(a.slots, 0, (int)(2u * a.P * kSlotBytes), 0x00020000);
  const G2Rsrc wr = g2_weights(a.qw, a.sc, a.zr, a.N, a.G), none = g2_weights(a.qw, a.sc, a.zr, a.N, a.G, false);
  const uint32_t row_bytes = (uint32_t)a.K * 2u;
  const int srow = 4 * (wave & 3) + (lane >> 4);   // row within the 16-row swizzle period
  const G2Rows rows{(uint32_t)(lane >> 4) * row_bytes + (uint32_t)((lane & 15) ^ srow) * 16u, row_bytes};
  constexpr bool kGlu = gemm_glu(OUT);
  using Op = std::conditional_t<OUT == GEMM_GLU16, G2F16, G2Bf16>;
  const int up = a.epi.up / kTileN;
  // groups [g0, g1) of tile t; stored if they are the whole tile
  auto segment = [&](int t, int g0, int g1) __attribute__((always_inline)) {
    int tn, tm;
    g2_tile_coords(a, t, tn, tm);
    const int m0 = tm * bm;
    const WaveTile w = g2_wave_tile<OUT>(a, tn, wt, b0);
    const int ltile = w.valid ? w.tile : (kGlu ? a.ld : a.N) / kTileN - 1;
    // Activation rows [m0, row end): the buffer's end turns rows past it into zeros.
    const uint16_t* A0 = a.A + (size_t)m0 * a.K;
    int norm[NH] = {};
    if constexpr (Op::kNorm) g2_load_norms<NH, kGlu>(norm, a.cexp, ltile, up, w.b0, lane);
    g2_segment<NH, NW, MB, kGlu, Op, 0>(a.G, norm, wr, none, g2_rsrc(A0, (uint32_t)(g2_row_end<NW>(a, m0) - m0) * row_bytes),
                                 g2_rsrc(A0, 0), rows, lds, acc, ltile, up, w.b0, mw, g0, g1, wave, lane);
    if (g0 != 0 || g1 != a.G) return false;
    if constexpr (OUT == GEMM_PLAIN) {
      g2_store_staged<NH, NW, MB>(a, acc, &lds[0][0], m0, w.tile, b0, mw, w.valid, wave, lane);
    } else {
      const size_t at = (size_t)m0 * a.ld + w.col;
      Epilogue e = a.epi;
      if (e.bias) e.bias += w.col;
      if (e.res) e.res += at;
      g2_store_epilogue<MB, kGlu, Op, 0>(acc, &lds[0][0], a.C + at, e, a.rexp + m0, a.cexp + w.col, a.ld,
                                         a.M - m0, w.valid, wave, lane);
    }
    return true;
  };
  for (int t = vp; t < a.full; t += a.P) segment(t, 0, a.G);
  for (int u = u0; u < u1;) {
    const int ts = u / a.G, g0 = u - ts * a.G;
    const int g1 = min(a.G, u1 - ts * a.G);
    if (!segment(a.full + ts, g0, g1)) g2_slot_store<NH, NW, MB>(rs, acc, vp, u == u0 ? 0 : 1, wave, lane);
    u = ts * a.G + g1;
  }
}

// Workspace bytes that enable stream-K: two fp32 partial tiles per CU.
size_t gemm_workspace_need(int cus) { return 2ull * (size_t)cus * kSlotBytes; }

// Tuning and test override of the prefill schedule (qw4_tune_gemm): -1 the
// cost model, 0 per tile, 1 stream-K, 2 hybrid, 3 split-K.
std::atomic<int> g_gemm_schedule{-1};
// Kernel variant (qw4_tune_gemm): 0 the default, 4 waves of whole 64-row
// tiles against all 256 activation rows; 1 8 waves of 32-row tile halves; 2 8
// waves of whole tiles against 128 rows. All three cut a call the same way and
// sum every output in the same order, so their results are bitwise equal.
std::atomic<int> g_gemm_variant{0};

template <int NH, int NW, int MB, int OUT = GEMM_PLAIN>
void launch_gemm(const GemmArgs& a, int grid, int nt, hipStream_t s) {
  k_gemm<NH, NW, MB, OUT><<<grid, 64 * NW, 0, s>>>(a);
  if (a.full != nt)   // the split tiles
    k_gemm_fixup<NH, NW, MB, OUT><<<(nt - a.full) * NW * G2Split<NH, NW, MB>::FIXP, 64, 0, s>>>(a);
}

template <int OUT>
void launch_gemm_rows(const GemmArgs& a, int mb, int grid, int nt, hipStream_t s) {
  switch (mb) {
    case 2: return launch_gemm<2, 4, 2, OUT>(a, grid, nt, s);
    case 3: return launch_gemm<2, 4, 3, OUT>(a, grid, nt, s);
    case 4: return launch_gemm<2, 4, 4, OUT>(a, grid, nt, s);
    case 5: return launch_gemm<2, 4, 5, OUT>(a, grid, nt, s);
    case 6: return launch_gemm<2, 4, 6, OUT>(a, grid, nt, s);
    case 7: return launch_gemm<2, 4, 7, OUT>(a, grid, nt, s);
    default: return launch_gemm<2, 4, 8, OUT>(a, grid, nt, s);
  }
}

// How a call is cut: tiles of 32 mb rows, schedule (0 per tile, 1 stream-K, 2
// hybrid, 3 split-K in S slices) and its cost.
struct GemmPlan {
  int mb, tiles_n, tiles_m, pick, S;
  double cost;
};

// Time of one (tile, group) step by its m-blocks, relative to 8. Measured over
// whole rounds of tiles (65536x5120, 256 and 1000 rows; us per 40 groups): 2 60,
// 3 74, 4 91, 5 101, 6 110, 7 125, 8 145; 2, 3, 6 and 7 are charged 5 to 20% more,
// for the memory latency that they expose when tiles are split. Over 12 projections
// x 12 row counts from 48 to 1500, timed at every height and schedule, the plan's
// pick is 1.3% (geometric mean) from the fastest; with the figures above as they
// are 1.2%, but up to 5% slower than 256-row tiles.
double step_cost(int mb) { return mb < 4 ? 0.38 + 0.06 * mb : 0.22 + 0.0975 * mb; }

GemmPlan gemm_plan(int M, int N, long long G, int mb, int cus, bool ws_ok, int schedule) {
  GemmPlan p{mb, (N + G2_BN - 1) / G2_BN, (M + 32 * mb - 1) / (32 * mb), 0, 0, 0.};
  const int nt = p.tiles_n * p.tiles_m, rem = nt % cus;
  // Schedules, costed in group-steps per CU (one tile x 128 step; measured on
  // MI355X at the config-4 shapes):
  //  * per tile: one workgroup per tile, ceil(nt / CUs) G;
  //  * stream-K: one workgroup per CU, all nt G (tile, group) units split
  //    evenly, nt G / CUs + 16 (two fp32 partial tiles written per
  //    workgroup) + 0.1 per piece of a cut tile (k_gemm_fixup's blocks read
  //    a tile's pieces one after another);
  //  * hybrid: whole tiles for the floor(nt / CUs) full rounds, then the
  //    other nt % CUs tiles split over the CUs: the same work, one partial
  //    per workgroup (+8), CUs / (nt % CUs) pieces per cut tile;
  //  * split-K (at most CUs / 2 tiles): every tile cut into the same S
  //    k-slices, S = CUs / nt (P = nt S workgroups, a multiple of 8, at
  //    least 4 groups per slice): G / S + 8 + 0.1 S. Against stream-K it
  //    writes one partial per workgroup instead of up to two, and the
  //    workgroups of an XCD share A at the same k (down M = 1024: 0.159
  //    against 0.170-0.180 ms; down M = 512 0.094 against 0.102-0.107).
  // A split schedule runs when it beats per-tile by 5% (qw4_tune_gemm
  // forces one, for tests and tuning): gate M = 512, 136 tiles, costs 37.6
  // against 40 and measured 0.880 against 0.842 PFLOP/s.
  const double t_dp = (double)((nt + cus - 1) / cus) * G;
  const double work = (double)nt * G / cus;
  const double t_sk = work + 16.0 + 0.1 * ((cus + nt - 1) / nt + 1);
  const double t_hy = work + 8.0 + 0.1 * (rem ? (cus + rem - 1) / rem + 1 : 0);
  ws_ok = ws_ok && rem != 0 && (long long)nt * G < (1LL << 31);
  const bool sk_ok = ws_ok && (long long)nt * G >= 2LL * cus;
  const bool hy_ok = ws_ok && nt > cus && (long long)rem * G >= (long long)cus;
  int S = 2 * nt <= cus ? (int)std::min<long long>(cus / nt, G >= 8 ? G / 4 : G / 2) : 0;
  while (S >= 2 && (nt * S) % 8) --S;
  const bool kk_ok = ws_ok && S >= 2;
  const double t_kk = (double)G / (S > 0 ? S : 1) + 8.0 + 0.1 * S;
  p.cost = t_dp;
  if (schedule == -1) {
    double best = 0.95 * t_dp;
    if (sk_ok && t_sk < best) { p.pick = 1; p.cost = best = t_sk; }
    if (hy_ok && t_hy < best) { p.pick = 2; p.cost = best = t_hy; }
    if (kk_ok && t_kk < best) { p.pick = 3; p.cost = t_kk; }
  } else if ((schedule == 1 && sk_ok) || (schedule == 2 && hy_ok) || (schedule == 3 && kk_ok)) {
    p.pick = schedule;
  }
  p.S = S;
  p.cost *= step_cost(mb);
  return p;
}

// Checked arguments; the epilogue of GEMM_PLAIN is empty.
template <int OUT>
int run_gemm(uint16_t* C, const qw4_weights* w, const uint16_t* A, int M, qw4_workspace* ws,
             const Epilogue& epi, void* stream) {
  // Loads address A and the weights through 32-bit buffer offsets.
  if ((size_t)M * w->in_f * 2 >= (1ull << 32) || (size_t)w->out_f * w->in_f / 2 >= (1ull << 32))
    return QW4_ERR_SHAPE;
  const int schedule = g_gemm_schedule.load(std::memory_order_relaxed);
  const int variant = OUT == GEMM_PLAIN ? g_gemm_variant.load(std::memory_order_relaxed) : 0;
  const int cus = device_cus();
  // fp16 operands at the end of the workspace, partial tiles at its start
  HalfRows half{};
  size_t space = ws && ws->buf ? ws->bytes & ~(size_t)255 : 0;
  if constexpr (OUT == GEMM_GLU16) {
    space -= half_rows_bytes(M, w);
    half = half_rows(static_cast<char*>(ws->buf) + space, A, M, w, (hipStream_t)stream);
    A = half.x;
  }
  const bool ws_ok = space >= gemm_workspace_need(cus) && cus % 8 == 0;
  GemmPlan p = gemm_plan(M, w->out_f, w->num_groups, 8, cus, ws_ok, schedule);
  // Tiles of fewer rows where that costs less: rows that do not fill 256-row
  // tiles (us, 256-row tiles against the plan's: gate|up 34816x5120 at 64 / 128 /
  // 300 rows 98 / 98 / 150 -> 55 / 70 / 126, down 5120x17408 53 / 55 / 87 -> 30 / 39 /
  // 66, o 5120x4096 36 / 36 / 40 -> 19 / 23 / 31), and few tiles, cut in fewer
  // slices (o at 256 rows 37 -> 28). By 3% at least, what the model resolves:
  // down at 2000 rows costs 100.9 in 224-row tiles against 101.3 and is 3% slower.
  // Stream-K and hybrid of lower tiles by 7% against 256 rows: the cost of a
  // workgroup's second segment does not shrink with the tile (9472x8448 at 500 / 1000
  // rows, 128-row tiles costed at 0.93 / 0.95 of 256-row ones: 96.7 / 164 us against
  // 94.0 / 155).
  if (schedule == -1) {
    const double cost8 = p.cost;
    for (int mb = 7; mb >= 2; --mb) {
      const GemmPlan q = gemm_plan(M, w->out_f, w->num_groups, mb, cus, ws_ok, schedule);
      if (q.cost < 0.97 * p.cost && !((q.pick == 1 || q.pick == 2) && q.cost >= 0.93 * cost8)) p = q;
    }
  }
  const int nt = p.tiles_n * p.tiles_m, mb = p.mb;
  GemmArgs a{w->qweight, w->scale, w->zeros, A, C, nullptr, M, w->out_f, w->in_f,
             w->num_groups, p.tiles_n, p.tiles_m, nt % 8 == 0, 32 * mb, nt, nt, 0,
             epi, gemm_glu(OUT) ? w->out_f / 2 : w->out_f, half.rexp, half.cexp};
  int grid = nt;
  if (p.pick == 3) {
    a.slots = static_cast<float*>(ws->buf);
    a.P = nt * p.S;
    a.full = 0;
    a.U = nt * w->num_groups;
    a.map = 2;
    grid = a.P;
  } else if (p.pick) {
    a.slots = static_cast<float*>(ws->buf);
    a.P = cus;
    a.full = p.pick == 2 ? nt - nt % cus : 0;
    a.U = (nt - a.full) * w->num_groups;
    a.map = 1;
    grid = cus;
  }
  hipStream_t s = (hipStream_t)stream;
  if constexpr (OUT == GEMM_PLAIN) {
    if (variant == 1)
      launch_gemm<1, 8, 8>(a, grid, nt, s);
    else if (variant == 2)
      launch_gemm<2, 8, 8>(a, grid, nt, s);
    else
      launch_gemm_rows<OUT>(a, mb, grid, nt, s);
  } else {
    launch_gemm_rows<OUT>(a, mb, grid, nt, s);
  }
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_workspace_alloc(qw4_workspace* ws, size_t bytes) {
  if (!ws) return QW4_ERR_NULL;
  std::memset(ws, 0, sizeof(*ws));
  if (bytes == 0) return QW4_OK;
  hipError_t e = hipMalloc(&ws->buf, bytes);
  if (e != hipSuccess) {
    set_hip_error((int)e);
    (void)hipGetLastError();
    ws->buf = nullptr;
    return QW4_ERR_NOMEM;
  }
  ws->bytes = bytes;
  return QW4_OK;
}

int qw4_workspace_free(qw4_workspace* ws) {
  if (!ws) return QW4_ERR_NULL;
  if (ws->buf) (void)hipFree(ws->buf);
  std::memset(ws, 0, sizeof(*ws));
  return QW4_OK;
}

int qw4_tune_gemm(int schedule, int variant) {
  if (schedule < -1 || schedule > 3 || variant < 0 || variant > 2) return QW4_ERR_SHAPE;
  g_gemm_schedule.store(schedule, std::memory_order_relaxed);
  g_gemm_variant.store(variant, std::memory_order_relaxed);
  return QW4_OK;
}

int qw4_gemm(uint16_t* C, const qw4_weights* w, const uint16_t* A, int M, qw4_workspace* ws,
             void* stream) {
  int st = check_weights_public(w);
  if (st) return st;
  if (!C || !A) return QW4_ERR_NULL;
  if (M < 1) return QW4_ERR_M;
  if (((uintptr_t)A & 15) || ((uintptr_t)C & 7)) return QW4_ERR_ALIGN;
  return run_gemm<GEMM_PLAIN>(C, w, A, M, ws, Epilogue{}, stream);
}

}  // extern "C"

int qw4::gemm_epilogue(uint16_t* y, const qw4_weights* w, const uint16_t* x, int M, qw4_workspace* ws,
                       const Epilogue& e, void* stream) {
  if (e.act != QW4_ACT_SWIGLU) return run_gemm<GEMM_EPI>(y, w, x, M, ws, e, stream);
  if (ws && ws->buf && ((uintptr_t)ws->buf & 255) == 0 && (size_t)M * w->in_f * 2 < (1ull << 32) &&
      (ws->bytes & ~(size_t)255) >= half_rows_bytes(M, w))
    return run_gemm<GEMM_GLU16>(y, w, x, M, ws, e, stream);
  return run_gemm<GEMM_GLU>(y, w, x, M, ws, e, stream);
}
