// The MFMA tile of the prefill GEMM, shared by the dense product (gemm.hip) and the
// products grouped by expert (grouped.hip): how a workgroup's waves load and
// dequantize their weights, stage activation rows in LDS, and multiply.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qwen_w4a16.h"
#include "epilogue.h"
#include "w4a16_common.h"

namespace qw4 {

// x in fp16 with an exponent a row, and an exponent for each weight row (k_half_rows).
struct HalfRows {
  const uint16_t* x;
  const int *rexp, *cexp;
};
// Bytes of a workspace that they take.
size_t half_rows_bytes(int T, const qw4_weights* w);
// Fills them, from buf on (half_rows.hip).
HalfRows half_rows(void* buf, const uint16_t* x, int T, const qw4_weights* w, hipStream_t s);


// ---------------------------------------------------------------------------
// k_gemm: 256 (M) x 256 (N) workgroup tile -- 32 MB (M) for MB = 2..7 m-blocks
// where the rows do not fill 256 (gemm_plan) -- v_mfma_f32_32x32x16_bf16 (the
// full-rate bf16 shape on gfx950). The default: 4 waves, one per SIMD, each a
// whole 64-row weight tile against all the tile's activation rows (its 32 MB
// accumulator registers in AGPRs); G2Split below lists the 8-wave forms.
//
//  * Weights are the MFMA A operand (rows = output columns n). Each wave loads
//    its packed rows straight into registers -- 32 B per lane per group, one
//    group ahead -- and dequantizes them in registers to exactly
//    RNE((q - z) * s): every weight element is converted once per workgroup
//    and never touches LDS.
//  * Activations are the B operand. A group's 256 x 128 activation tile goes
//    global -> LDS directly (global_load_lds_dwordx4), double-buffered, one
//    instruction per 4 full rows (1 KiB, fully coalesced). LDS row m holds
//    16-byte chunk c of the row at slot c ^ (m % 16): lane i of a load
//    instruction writes slot i % 16 and so fetches chunk (i % 16) ^ (m % 16)
//    (the XOR keeps each 4-lane group inside one 64-byte sector). The MFMA
//    operand reads (32 rows x 16 B per half-wave) then hit distinct banks.
//  * k permutation: lane l (row r = l % 32, half h = l / 32) of k-step (s, t)
//    holds k = 64 s + 32 h + 8 t + e -- word t of chunk 2 s + h of its weight
//    row -- and reads the activation chunk 8 s + 4 h + t, the same k.
//  * Row permutation: MFMA row r of tile half b reads tile position
//    p = 16 (r % 4) + 8 b + 2 (r / 8) + (r / 4) % 2, so the four D rows a lane
//    holds for each r / 8 are four consecutive output columns (an 8-byte
//    piece of a staged row, see g2_store_staged).
constexpr int G2_BM = 256, G2_BN = 256;   // rows at most (32 MB of them, see G2Split), columns

typedef float f32x16v __attribute__((ext_vector_type(16)));

// Work split of a workgroup's 4 weight tiles x 8 m-blocks over its NW waves:
//  * NH = 1, NW = 8: a wave owns one 32-row tile half against all 8 m-blocks;
//  * NH = 2, NW = 8: a wave owns a whole 64-row tile against 4 m-blocks (half
//    the LDS reads per MFMA, every weight dequantized by two waves);
//  * NH = 2, NW = 4: one wave per SIMD owns a whole tile against all 8
//    m-blocks (half the LDS reads, every weight dequantized once; its 256
//    accumulator registers take the AGPR half of the register file).
// MB: 32-row m-blocks of the workgroup's tile, 8 unless fewer rows need it.
// DD: groups buffered, 0 for as many as the CU's LDS holds.
template <int NH, int NW, int MB, int DD = 0>
struct G2Split {
  static constexpr int MBW = 8 * MB / (NW * NH);     // m-blocks per wave
  static constexpr int UNITS = NH * MBW;             // (half, m-block) pairs per wave
  static constexpr int ACT = 8 * MB / NW;            // 1 KiB (4-row) activation loads per wave and group
  static constexpr int FIXP = (UNITS + 1) / 2;       // fixup blocks per wave region
  // groups buffered: as many 8 MB KiB activation buffers as LDS holds, 4 at most
  // (MB = 5: three buffers spill 17 VGPRs, 72 bytes a lane, and are still faster
  // than two without a spill: whole tiles 3%, split-K 1%, the others equal)
  static constexpr int DEPTH = DD ? DD : MB <= 4 ? 4 : MB == 5 ? 3 : 2;
  // k-step schedule (measured on MI355X at the config-4 shapes): VALU slots
  // after each MFMA, LDS operand reads after each of the first MFMAs, and the
  // k-steps that carry the next group's activation loads.
  static constexpr int VALU = NW == 8 ? 4 * NH : 2;
  static constexpr int DS = 2;
  static constexpr int ACTSTEPS = NW == 8 ? 4 : 8;
  static_assert(MBW * NH * NW == 8 * MB && ACT * NW == 8 * MB, "unsupported split");
  __device__ static void coords(int wave, int& wt, int& b0, int& mw) {
    wt = NH == 1 ? (wave >> 1) : (wave & 3);   // tile of the 4 this wave owns
    b0 = NH == 1 ? (wave & 1) : 0;             // first tile half
    mw = NH == 1 ? 0 : (wave >> 2) * MBW;      // first m-block
  }
};

template <int NH>
struct WeightGroup {
  u32x4 q[NH][2];    // [half][s]: chunk 2 s + h of this lane's weight row
  uint32_t s[NH];    // scale bits
  uint32_t z[NH];    // zero-point word (4 rows, 4 bits each)
};

// Buffer-resource addressing: a 32-bit per-lane offset (loop-invariant) plus
// a scalar offset, instead of a 64-bit address per lane and load. Loads are
// unconditional (an out-of-range wave reads the last tile and stores nothing),
// and the zero-point word is kept raw: arithmetic on a loaded value here
// would make the compiler wait for every earlier load, including the
// activation loads just issued.
struct G2Rsrc {
  __amdgpu_buffer_rsrc_t qw, sc, zr;
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t g2_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
// The weights of N rows x G groups; of no length without some.
__device__ __forceinline__ G2Rsrc g2_weights(const uint32_t* qw, const uint16_t* sc, const uint16_t* zr,
                                             int N, int G, bool some = true) {
  const uint32_t blocks = some ? (uint32_t)N / kTileN * (uint32_t)G : 0u;
  return {g2_rsrc(qw, blocks * 4096u), g2_rsrc(sc, blocks * (uint32_t)kMetaBytes), g2_rsrc(zr, blocks * 32u)};
}

// The exponents of a lane's weight rows (part j as in g2_load_weights), cexp [N].
template <int NH, bool GLU>
__device__ __forceinline__ void g2_load_norms(int (&norm)[NH], const int* cexp, int tile, int up, int b0,
                                              int lane) {
  const int r = lane & 31;
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    const int a16 = 8 * (GLU ? b0 : b0 + j) + 2 * (r >> 3) + ((r >> 2) & 1);
    norm[j] = cexp[(GLU ? tile + j * up : tile) * kTileN + 4 * a16 + (r & 3)];
  }
}

// part j < NH: the packed words of part j; part NH: the scales and zero
// points; part -1: everything. Part j is half b0 + j of the tile; in a gated
// product (GLU) half b0 of the gate tile (j = 0) or of its up tile, `up` tiles on.
template <int NH, bool GLU = false>
__device__ __forceinline__ void g2_load_weights(WeightGroup<NH>& wg, const G2Rsrc& rs, int G,
                                                int tile, int up, int b0, int g, int lane,
                                                int part = -1) {
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    const uint32_t blk = (uint32_t)(GLU ? tile + j * up : tile) * (uint32_t)G + (uint32_t)g;   // < 2^26
    const int a16 = 8 * (GLU ? b0 : b0 + j) + 2 * (r >> 3) + ((r >> 2) & 1);   // position % 16
    const int p = 16 * (r & 3) + a16;
    if (part < 0 || part == j) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        wg.q[j][s] = __builtin_amdgcn_raw_buffer_load_b128(rs.qw, ((2 * s + h) * 64 + p) * 16,
                                                           blk * 4096u, 0);
    }
    if (part < 0 || part == NH) {
      wg.s[j] = __builtin_amdgcn_raw_buffer_load_b16(rs.sc, (4 * a16 + (r & 3)) * 2, blk * (uint32_t)kMetaBytes, 0);
      wg.z[j] = __builtin_amdgcn_raw_buffer_load_b16(rs.zr, a16 * 2, blk * 32u, 0);
    }
  }
}

// Byte offset of a lane's 16 bytes in activation load i of its wave (row block rb =
// i NW + wave: 4 rows, 1 KiB). Rows in a run: voff is the lane's offset in the first
// row block; the swizzle repeats every 4 blocks, so it is the same for all of a
// wave's. Rows gathered by an index: an offset per load.
struct G2Rows {
  uint32_t voff, row_bytes;
  __device__ uint32_t at(int, int rb) const { return voff + (uint32_t)(4 * rb) * row_bytes; }
};
template <int N>
struct G2Gather {
  uint32_t off[N];
  __device__ uint32_t at(int i, int) const { return off[i]; }
};

__device__ __forceinline__ void g2_load_lds16(__amdgpu_buffer_rsrc_t r, u32x4* dst, uint32_t voff,
                                              uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, dst, 16, voff, soff, 0, 0);
}

// Issue activation load i of group g into buf. Rows outside `act` read as zeros.
template <int NW, class Rows>
__device__ __forceinline__ void g2_load_act1(__amdgpu_buffer_rsrc_t act, const Rows& rows, u32x4* buf,
                                             int g, int wave, int i) {
  const int rb = i * NW + wave;
  g2_load_lds16(act, buf + rb * 64, rows.at(i, rb), (uint32_t)g * (kGroup * 2));
}

// One packed word -> 8 bf16 weights RNE((q - z) s), c = -z s, in the order
// of nib8_bits (register i: elements i and i + 4). The even nibbles are the
// low nibbles of the bytes of w & 0x0F0F0F0F, the odd ones of (w >> 4): each
// converts to fp32 in one v_cvt_f32_ubyteN, and fma(q, s, -z s) is exact
// (both products have at most 12 significant bits) -- 23 VALU per word.
__device__ __forceinline__ bf16x8 g2_deq(uint32_t w, float s, float c) {
  const uint32_t ev = w & 0x0F0F0F0Fu, od = (w >> 4) & 0x0F0F0F0Fu;
  float q[8];   // q[2 b] = byte b of ev, q[2 b + 1] = byte b of od
  asm("v_cvt_f32_ubyte0 %0, %1" : "=v"(q[0]) : "v"(ev));
  asm("v_cvt_f32_ubyte1 %0, %1" : "=v"(q[2]) : "v"(ev));
  asm("v_cvt_f32_ubyte2 %0, %1" : "=v"(q[4]) : "v"(ev));
  asm("v_cvt_f32_ubyte3 %0, %1" : "=v"(q[6]) : "v"(ev));
  asm("v_cvt_f32_ubyte0 %0, %1" : "=v"(q[1]) : "v"(od));
  asm("v_cvt_f32_ubyte1 %0, %1" : "=v"(q[3]) : "v"(od));
  asm("v_cvt_f32_ubyte2 %0, %1" : "=v"(q[5]) : "v"(od));
  asm("v_cvt_f32_ubyte3 %0, %1" : "=v"(q[7]) : "v"(od));
  auto f = [&](int e) { return __builtin_fmaf(q[e], s, c); };
  u32x4 o;
  o[0] = pack_bf16x2(f(0), f(4));   // elements 0, 4 (bytes 0 and 2 of ev)
  o[1] = pack_bf16x2(f(1), f(5));   // 1, 5
  o[2] = pack_bf16x2(f(2), f(6));   // 2, 6
  o[3] = pack_bf16x2(f(3), f(7));   // 3, 7
  return __builtin_bit_cast(bf16x8, o);
}

// The two operand types of the tile.
//  * G2Bf16: activations as they are, weights RNE((q - z) s) to bf16 (8 bits), the
//    reference's arithmetic.
//  * G2F16: weights to 11 bits, RNE((q - z) s 2^-e), e the exponent of their row's
//    largest scale, and activation rows times a power of two that brings their largest
//    value to 2^14 (k_half_rows); exact in fp16 but for what lies 2^-28 (a scale: 2^-20)
//    below its row's largest. The sums take the exponents back in the epilogue. For gated
//    products, whose factors each carry the weights' rounding: 0.0027 of the output's
//    rms in bf16, 0.0017 (the output's own rounding) so; and for ungated ones by expert
//    where qw4_linear would use a weight of the expert's size exactly (0.0022, 0.0017).
struct G2Bf16 {
  static constexpr bool kNorm = false;
  struct Scale {
    float s, c;
  };
  __device__ static Scale scale(uint32_t s, uint32_t z, int) {
    const float sf = bf16_bits_to_f32(s);
    return {sf, -(float)z * sf};
  }
  __device__ static bf16x8 deq(uint32_t w, const Scale& k) { return g2_deq(w, k.s, k.c); }
  __device__ static f32x16v mfma(bf16x8 a, u32x4 b, f32x16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

struct G2F16 {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  static constexpr bool kNorm = true;
  // pairs of s 2^-e and of -(1024 + z) for even nibbles, of s 2^-e / 16 and of
  // -(1024 + 16 z) for odd ones
  struct Scale {
    uint32_t s, z, s16, z16;
  };
  __device__ static Scale scale(uint32_t s, uint32_t z, int e) {
    const _Float16 h = (_Float16)__builtin_ldexpf(bf16_bits_to_f32(s), -e);
    const _Float16 h16 = (_Float16)__builtin_ldexpf(bf16_bits_to_f32(s), -e - 4);
    return {__builtin_bit_cast(uint32_t, f16x2{h, h}), (z * 0x10001u) | 0xE400E400u,
            __builtin_bit_cast(uint32_t, f16x2{h16, h16}), (z * 0x100010u) | 0xE400E400u};
  }
  // A nibble in the low four mantissa bits of 1024 is 1024 + q, in the next four 1024 + 16 q;
  // less 1024 + z or 1024 + 16 z it is exact, and the product with the scale rounds once:
  // 13 VALU per word (15 with each nibble shifted down: 1% slower, 3% on tiles of 64 rows).
  __device__ static bf16x8 deq(uint32_t w, const Scale& k) {
    const f16x2 s = __builtin_bit_cast(f16x2, k.s), z = __builtin_bit_cast(f16x2, k.z);
    const f16x2 s16 = __builtin_bit_cast(f16x2, k.s16), z16 = __builtin_bit_cast(f16x2, k.z16);
    // the constants in registers, for one v_and_or_b32 a pair (see NibConst)
    uint32_t low, high, magic;
    asm("v_mov_b32 %0, 0x000f000f" : "=v"(low));
    asm("v_mov_b32 %0, 0x00f000f0" : "=v"(high));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(magic));
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t v = w >> (4 * i);
      const f16x2 even = __builtin_bit_cast(f16x2, (v & low) | magic);
      const f16x2 odd = __builtin_bit_cast(f16x2, (v & high) | magic);
      o[i] = __builtin_bit_cast(uint32_t, (even + z) * s);
      o[i + 1] = __builtin_bit_cast(uint32_t, (odd + z16) * s16);
    }
    return __builtin_bit_cast(bf16x8, o);   // the bits; mfma takes them as fp16
  }
  __device__ static f32x16v mfma(bf16x8 a, u32x4 b, f32x16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b),
                                                  c, 0, 0, 0);
  }
};

// s_waitcnt vmcnt(0) (expcnt and lgkmcnt left at their maxima).
__device__ __forceinline__ void g2_wait_vm0() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// Workgroups are dealt round-robin to the 8 XCDs (each with its own L2): XCD x
// runs blocks x, x + 8, ... Renumber so that each XCD owns a contiguous run of
// work. Needs count % 8 == 0 (then it is a bijection).
__device__ __forceinline__ int g2_xcd_order(int blk, int count) {
  return (blk & 7) * (count >> 3) + (blk >> 3);
}

// One group of a segment: the MFMAs of group g (its activation rows in buf, its
// weights in cur) while the loads of a later group gn go out, activations into
// nbuf and weights into nxt (actn, rsn: zero-length resources where there is no
// such group -- they fetch nothing and need no branch, which would split the
// k-step schedule).
// norm: G2F16's exponents of the lane's weight rows.
template <int NH, int NW, int MB, bool GLU, class Op, class Rows>
__device__ __forceinline__ void g2_group(int G, const int (&norm)[NH],
                                         f32x16v (&acc)[NH][G2Split<NH, NW, MB>::MBW],
                                         const WeightGroup<NH>& cur, WeightGroup<NH>& nxt,
                                         const u32x4* buf, u32x4* nbuf,
                                         __amdgpu_buffer_rsrc_t actn, const G2Rsrc& rsn,
                                         const Rows& rows, int ltile, int up, int b0, int gn,
                                         int wave, int lane) {
  using Sp = G2Split<NH, NW, MB>;
  constexpr int MBW = Sp::MBW;
  const int r = lane & 31, h = lane >> 5;
  const int zsh = 4 * (r & 3);
  // Group gn's activation rows spread evenly over the first Sp::ACTSTEPS
  // k-steps below, so that what the workgroup writes into LDS per group does
  // not arrive in one burst on top of the first steps' operand reads (8
  // waves: steps 0-3, 4% faster than one burst and 1.5% than one load per
  // step; 4 waves: all 8 steps, equal to steps 0-3); its weights in k-steps
  // kWStep.. kWStep + NH (0.5-0.8% faster than all at the group's start, where
  // they delay its first MFMA).
  typename Op::Scale sc[NH];
#pragma unroll
  for (int j = 0; j < NH; ++j) sc[j] = Op::scale(cur.s[j], (cur.z[j] >> zsh) & 0xFu, norm[j]);
  // Software pipeline over the group's 8 k-steps: the activation operands
  // and the dequantized weight operands of step u + 1 are produced while
  // step u's MFMAs run.
  u32x4 xo[2][MBW];
  bf16x8 wd[2][NH];
#pragma unroll
  for (int mb = 0; mb < MBW; ++mb) xo[0][mb] = buf[mb * 512 + ((4 * h) ^ (r & 15))];
#pragma unroll
  for (int j = 0; j < NH; ++j) wd[0][j] = Op::deq(cur.q[j][0][0], sc[j]);
  // Fence: the prologue's reads must not fill the DS slots of the pattern below.
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int cu = u & 1, nu = cu ^ 1;
    constexpr int kWStep = 4;
    if (u >= kWStep && u <= kWStep + NH)
      g2_load_weights<NH, GLU>(nxt, rsn, G, ltile, up, b0, gn, lane, u - kWStep);
    if (u < Sp::ACTSTEPS) {
#pragma unroll
      for (int i = Sp::ACT * u / Sp::ACTSTEPS; i < Sp::ACT * (u + 1) / Sp::ACTSTEPS; ++i)
        g2_load_act1<NW>(actn, rows, nbuf, gn, wave, i);
    }
    if (u + 1 < 8) {
      const int s1 = (u + 1) >> 2, t1 = (u + 1) & 3;
      const int slot = (8 * s1 + 4 * h + t1) ^ (r & 15);
#pragma unroll
      for (int mb = 0; mb < MBW; ++mb) xo[nu][mb] = buf[mb * 512 + slot];
#pragma unroll
      for (int j = 0; j < NH; ++j) wd[nu][j] = Op::deq(cur.q[j][s1][t1], sc[j]);
    }
#pragma unroll
    for (int mb = 0; mb < MBW; ++mb)
#pragma unroll
      for (int j = 0; j < NH; ++j)
        acc[j][mb] = Op::mfma(wd[cu][j], xo[cu][mb], acc[j][mb]);
    if (u + 1 < 8) {
#pragma unroll
      for (int i = 0; i < MBW * NH; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        if (i < (MBW + Sp::DS - 1) / Sp::DS) __builtin_amdgcn_sched_group_barrier(0x100, Sp::DS, 0);  // DS read
        __builtin_amdgcn_sched_group_barrier(0x002, Sp::VALU, 0);  // VALU
      }
    }
    // NW = 4: one scheduling region per k-step, so that the next step's
    // operand reads stay under this step's MFMAs instead of sinking to their
    // first use (with one wave per SIMD nothing else hides their latency).
    if (NW == 4) __builtin_amdgcn_sched_barrier(0);
  }
}

// One wave's share of one (tile, group range) segment: acc = sum over groups
// [g0, g1) of this wave's weight rows x the tile's activation rows, which `rows`
// finds in `act`. rs_none, act_none: the same of no length, for the loads past the
// last group.
template <int NH, int NW, int MB, bool GLU, class Op, int DD, class Rows>
__device__ __forceinline__ void g2_segment(int G, const int (&norm)[NH], const G2Rsrc& rs, const G2Rsrc& rs_none,
                                           __amdgpu_buffer_rsrc_t act,
                                           __amdgpu_buffer_rsrc_t act_none, const Rows& rows, u32x4 (*lds)[32 * MB * 16],
                                           f32x16v (&acc)[NH][G2Split<NH, NW, MB>::MBW], int ltile,
                                           int up, int b0, int mw, int g0, int g1, int wave, int lane) {
  using Sp = G2Split<NH, NW, MB, DD>;
  constexpr int MBW = Sp::MBW, D = Sp::DEPTH;
  const int r = lane & 31;
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int mb = 0; mb < MBW; ++mb) acc[j][mb] = f32x16v{};
  __syncthreads();   // the previous segment's last LDS reads are done
  if constexpr (D == 2) {
    WeightGroup<NH> cur, nxt;
#pragma unroll
    for (int i = 0; i < Sp::ACT; ++i) g2_load_act1<NW>(act, rows, lds[0], g0, wave, i);
    g2_load_weights<NH, GLU>(cur, rs, G, ltile, up, b0, g0, lane);
    for (int g = g0; g < g1; ++g) {
      g2_wait_vm0();
      __syncthreads();
      const int sb = (g - g0) & 1;
      const bool more = g + 1 < g1;
      g2_group<NH, NW, MB, GLU, Op>(G, norm, acc, cur, nxt, lds[sb] + (32 * mw + r) * 16, lds[sb ^ 1],
                                more ? act : act_none, more ? rs : rs_none, rows, ltile, up, b0,
                                g + 1, wave, lane);
      cur = nxt;
    }
  } else {
    // D buffers, the loads D - 1 groups ahead: a group of few m-blocks computes
    // in less than a memory latency. Unrolled by D, so that every buffer --
    // LDS and weight registers -- is named statically and no register is
    // copied (a copy would wait for its load). Waits are counted: loads
    // complete in order, and every group issues the same number.
    constexpr int kLoads = Sp::ACT + 4 * NH;
    WeightGroup<NH> wg[D];
#pragma unroll
    for (int d = 0; d < D - 1; ++d) {
      const bool in = g0 + d < g1;
#pragma unroll
      for (int i = 0; i < Sp::ACT; ++i)
        g2_load_act1<NW>(in ? act : act_none, rows, lds[d], g0 + d, wave, i);
      g2_load_weights<NH, GLU>(wg[d], in ? rs : rs_none, G, ltile, up, b0, g0 + d, lane);
    }
    for (int gb = g0; gb < g1; gb += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int g = gb + d;
        if (g >= g1) break;
        // group g has landed (the D - 2 groups behind it may be in flight) for
        // every wave, and every wave is done with group g - 1's buffer
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 2) * kLoads) : "memory");
        constexpr int kBack = D - 1;
        const bool more = g + kBack < g1;
        g2_group<NH, NW, MB, GLU, Op>(G, norm, acc, wg[d], wg[(d + kBack) % D], lds[d] + (32 * mw + r) * 16,
                                  lds[(d + kBack) % D], more ? act : act_none, more ? rs : rs_none,
                                  rows, ltile, up, b0, g + kBack, wave, lane);
      }
    }
  }
}

// Tile store with an epilogue. The accumulators go through LDS as fp32, as many
// m-blocks at a time as the wave's share of the activation buffers holds (its rows x
// 64 values: gate and up columns apart in a gated product; 16-byte chunk c of a row
// at c ^ (row % 16)), and come back row by row, 8 output columns a lane, so that bias
// and residual are added and the result rounded once, in whole 128-byte (gated: 64-byte)
// segments of a row. out and e.res point to the tile's first row and the wave's first
// column, e.bias to that column; `rows` rows are stored. G2F16: rexp are the exponents
// of the tile's rows, cexp those of the wave's columns (up columns e.up on).
template <int MB, bool GLU, class Op, int DD>
__device__ __forceinline__ void g2_store_epilogue(const f32x16v (&acc)[2][MB], u32x4* lds, uint16_t* out,
                                                  const Epilogue& e, const int* rexp, const int* cexp,
                                                  int ld, int rows, bool valid, int wave, int lane) {
  constexpr int kPass = G2Split<2, 4, MB, DD>::DEPTH * MB / 4;   // m-blocks of 8 KiB in a wave's share
  constexpr int kLanes = GLU ? 4 : 8;                        // lanes of a row, 8 columns each
  constexpr int kStep = 64 / kLanes;                         // rows of one instruction
  constexpr int kBatch = 32 / kStep;                         // residual loads in flight: an m-block's
  const int r = lane & 31, h = lane >> 5, cl = lane % kLanes, rl = lane / kLanes;
  g2_wait_vm0();
  __syncthreads();
  u32x4* reg = lds + wave * (kPass * 512);
  float bias[GLU ? 2 : 1][8];
  if (valid) load_bias<GLU>(bias, e, 8 * cl);
  int ce[GLU ? 2 : 1][8];
#pragma unroll
  for (int j = 0; j < (GLU ? 2 : 1); ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) ce[j][i] = Op::kNorm && valid ? cexp[j * e.up + 8 * cl + i] : 0;
#pragma unroll
  for (int p0 = 0; p0 < MB; p0 += kPass) {
    const int blocks = p0 + kPass <= MB ? kPass : MB - p0;
#pragma unroll
    for (int k = 0; k < kPass; ++k) {
      if (p0 + k >= MB) break;
      const int row = 32 * k + r;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int jq = 0; jq < 4; ++jq) {
          const f32x16v& v = acc[j][p0 + k < MB ? p0 + k : 0];
          reg[row * 16 + ((8 * j + 2 * jq + h) ^ (row & 15))] =
              u32x4{__float_as_uint(v[4 * jq]), __float_as_uint(v[4 * jq + 1]),
                    __float_as_uint(v[4 * jq + 2]), __float_as_uint(v[4 * jq + 3])};
        }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    if (valid) {
      for (int t0 = 0; t0 < 32 * blocks; t0 += kBatch * kStep) {
        u32x4 res[kBatch];
        int re[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int m = 32 * p0 + t0 + i * kStep + rl;
          res[i] = u32x4{0u, 0u, 0u, 0u};
          re[i] = Op::kNorm && m < rows ? rexp[m] : 0;
          if (e.res && m < rows) res[i] = *reinterpret_cast<const u32x4*>(e.res + (size_t)m * ld + 8 * cl);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int row = t0 + i * kStep + rl, m = 32 * p0 + row;
          float v[GLU ? 2 : 1][8];
#pragma unroll
          for (int j = 0; j < (GLU ? 2 : 1); ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const u32x4 w = reg[row * 16 + ((8 * j + 2 * cl + c) ^ (row & 15))];
#pragma unroll
              for (int i2 = 0; i2 < 4; ++i2) {
                float f = __uint_as_float(w[i2]);
                if (Op::kNorm) f = __builtin_ldexpf(f, re[i] + ce[j][4 * c + i2]);
                v[j][4 * c + i2] = f + bias[j][4 * c + i2];
              }
            }
          epilogue_act<GLU>(v, e.act);
          if (m < rows) *reinterpret_cast<u32x4*>(out + (size_t)m * ld + 8 * cl) = add_round8(v[0], res[i]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
}

}  // namespace qw4
