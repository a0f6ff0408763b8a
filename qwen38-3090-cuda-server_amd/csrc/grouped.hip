// W4A16 products grouped by expert: rows [offsets[e], offsets[e + 1]) of y are f(x_row
// W_e^T + b_e), the experts' weights stacked in one W4A16 tensor, x in the plan's order
// or gathered by its tokens. The row counts live on the device only: every workgroup
// reads the offsets and finds its own work, so that no call waits for the host and a
// captured graph routes anew on every replay.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/qwen_w4a16.h"
#include "gemm_tile.h"
#include "grouped.h"
#include "skinny.h"
#include "w4a16_common.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);

namespace {

// Many rows an expert: the MFMA tile of the prefill GEMM (gemm_tile.h) over (expert, row
// block, column tile). First the tiles of whole row blocks, expert by expert in bands of
// four blocks (a column tile's four together), then those of the blocks that experts end
// with, which compute a half or a quarter of the tile where that covers their rows, the
// shorter ones last. Rounds of P tiles go over the workgroups back and forth, so that
// who had a long one gets a short one; an XCD takes a run of a round, so that weights
// and rows stay in its L2.
//
// LDS for groups of M m-blocks: 8 M KiB each, up to four.
template <int MB, int DD>
constexpr int tile_depth(int m) {
  return MB * DD / m < 4 ? MB * DD / m : 4;
}

// Heights of an ending block: the whole tile, a half, at MB = 8 also a quarter.
template <int MB>
constexpr int tile_ends() {
  return MB >= 8 ? 3 : 2;
}

template <int MB, int DD, int OCC, bool GLU, bool GATHER, class Op>
__global__ __launch_bounds__(256, OCC) void k_grouped_tiles(GroupedArgs a) {
  // One LDS object for everything: of several, the compiler tells their accesses apart
  // and waits for all loads into one before it reads the next (vmcnt(0) at every k-step;
  // 32768 rows of 64 experts, 2048 x 2048: 339 us instead of 258).
  constexpr int kBufs = DD * 32 * MB * 16, kRows = GATHER ? 32 * MB : 0;
  constexpr int kEnds = tile_ends<MB>(), kLists = 1 + kEnds;
  __shared__ u32x4 lds[kBufs + (4 * kRows + kLists * (kMaxExperts + 1 + 4) + 3) / 4];
  // gathered rows: x's row and its exponent at each of the tile's positions, in turns:
  // a buffer is filled again a barrier after every wave is done with it
  int* const from = reinterpret_cast<int*>(lds + kBufs);
  int* const rexp = from + 2 * kRows;
  int* const start = rexp + 2 * kRows;
  int* const wsum = start + kLists * (kMaxExperts + 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int blocks[kLists];   // whole, and ending by height
  expert_starts<256>(a, start, wsum, blocks, [](int rows, int which) {
    const int end = rows % (32 * MB);
    // height 32 MB >> (which - 1): above the next lower one, if there is one
    const int high = 32 * MB >> (which - 1), low = which == kEnds ? 0 : high >> 1;
    return which == 0 ? rows / (32 * MB) : (int)(end > low && end <= high);
  });
  long long tiles = 0;
#pragma unroll
  for (int l = 0; l < kLists; ++l) tiles += (long long)blocks[l] * a.tiles_n;
  const int all = (int)min(tiles, 0x3fffffffLL);   // more: offsets of no plan
  const uint32_t row_bytes = (uint32_t)a.K * 2u;
  const int up = a.epi.up / kTileN;
  const int width = GLU ? a.ld : a.n;   // columns the column tiles run over
  int turn = 0;
  const int vp = a.P % 8 ? (int)blockIdx.x : (int)((blockIdx.x & 7) * (a.P >> 3) + (blockIdx.x >> 3));
  for (int base = 0, round = 0; base < all; base += a.P, ++round) {
    // the last round in launch order: its tiles spread over the XCDs and CUs
    int t = base + (base + a.P > all ? (int)blockIdx.x : round & 1 ? a.P - 1 - vp : vp);
    if (t >= all) continue;
    int list = 0;
    while (list + 1 < kLists && t >= blocks[list] * a.tiles_n) t -= blocks[list++] * a.tiles_n;
    const int* const first = start + list * (kMaxExperts + 1);
    const int e = expert_of(first, a.E, a.tiles_n, t);
    int lo, hi;
    expert_rows(a, e, lo, hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int n_whole = (hi - lo) / (32 * MB);
    const int at = t - __builtin_amdgcn_readfirstlane(first[e]) * a.tiles_n;
    if ((uint32_t)at >= (uint32_t)((list ? 1 : n_whole) * a.tiles_n)) continue;   // offsets of no plan
    int tn = at, block = n_whole;
    if (list == 0) {
      const int band = at / (4 * a.tiles_n), in_band = at - band * 4 * a.tiles_n;
      const int high = min(4, n_whole - 4 * band);
      tn = in_band / high;
      block = 4 * band + in_band - tn * high;
    }
    const int m0 = lo + block * 32 * MB;
    const int rows = hi - m0;
    // a wave's weight tile, half and first output column, as the dense product's
    const int wt = GLU ? tn * 2 + (wave >> 1) : tn * 4 + wave;
    const int b0 = GLU ? wave & 1 : 0;
    const int col = wt * kTileN + 32 * b0;
    const bool valid = wt * kTileN < width;
    // opaque, so that the addresses of every height are formed where they are used and
    // not kept, spilled, from before the loop
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int srow = 4 * wave + (lane >> 4);   // row within the 16-row swizzle period
    const uint32_t chunk = (uint32_t)((lane & 15) ^ srow) * 16u;
    const int ltile = valid ? wt : width / kTileN - 1;
    const size_t blk = (size_t)e * (a.n / kTileN) * a.G;   // the expert's first weight block
    const G2Rsrc wr = g2_weights(a.qw + blk * kWordsPerBlock, a.sc + blk * kMetaU16, a.zr + blk * 16, a.n, a.G);
    const G2Rsrc none =
        g2_weights(a.qw + blk * kWordsPerBlock, a.sc + blk * kMetaU16, a.zr + blk * 16, a.n, a.G, false);
    const int* cexp = Op::kNorm ? a.cexp + (size_t)e * a.n : nullptr;
    int norm[2] = {};
    if constexpr (Op::kNorm) g2_load_norms<2, GLU>(norm, cexp, ltile, up, b0, lane);
    turn ^= 1;
    if constexpr (GATHER) {
      for (int r = threadIdx.x; r < 32 * MB; r += 256) {
        const int row = r < rows ? a.tokens[m0 + r] : -1;
        from[turn * kRows + r] = row;
        if (Op::kNorm) rexp[turn * kRows + r] = (uint64_t)(uint32_t)row * row_bytes < a.x_bytes ? a.rexp[row] : 0;
      }
      __syncthreads();
    }
    Epilogue ep = a.epi;
    if (ep.bias) ep.bias += (size_t)e * a.n + col;
    auto tile = [&](auto mc) __attribute__((always_inline)) {
      constexpr int M = decltype(mc)::value, D = tile_depth<MB, DD>(M);
      constexpr int kAct = G2Split<2, 4, M, D>::ACT;
      f32x16v acc[2][M];
      auto* const buf = reinterpret_cast<u32x4(*)[32 * M * 16]>(lds);
      if constexpr (GATHER) {
        G2Gather<kAct> g;
#pragma unroll
        for (int i = 0; i < kAct; ++i) {
          // past the block, or past x: reads as zeros
          const uint64_t off = (uint64_t)(uint32_t)from[turn * kRows + 4 * (4 * i + wave) + (lane >> 4)] * row_bytes;
          g.off[i] = off < a.x_bytes ? (uint32_t)off + chunk : a.x_bytes;
        }
        g2_segment<2, 4, M, GLU, Op, D>(a.G, norm, wr, none, g2_rsrc(a.x, a.x_bytes), g2_rsrc(a.x, 0), g, buf,
                                        acc, ltile, up, b0, 0, 0, a.G, wave, lane);
      } else {
        const uint16_t* x0 = a.x + (size_t)m0 * a.K;
        const G2Rows g{(uint32_t)(lane >> 4) * row_bytes + chunk, row_bytes};
        g2_segment<2, 4, M, GLU, Op, D>(a.G, norm, wr, none, g2_rsrc(x0, (uint32_t)min(rows, 32 * M) * row_bytes),
                                        g2_rsrc(x0, 0), g, buf, acc, ltile, up, b0, 0, 0, a.G, wave, lane);
      }
      const int* re = !Op::kNorm ? nullptr : GATHER ? rexp + turn * kRows : a.rexp + m0;
      g2_store_epilogue<M, GLU, Op, D>(acc, lds, a.y + (size_t)m0 * a.ld + col, ep, re, cexp + col, a.ld, rows,
                                       valid, wave, lane);
    };
    if (list <= 1)
      tile(std::integral_constant<int, MB>{});
    else if (kEnds == 2 || list == 2)
      tile(std::integral_constant<int, MB / 2>{});
    else
      tile(std::integral_constant<int, MB / (kEnds == 3 ? 4 : 2)>{});
  }
}

std::atomic<int> g_form{0};   // qw4_tune_grouped

template <int MB, int DD, int OCC, bool GLU, class Op>
void launch_tiles(const GroupedArgs& a, hipStream_t s) {
  a.tokens ? k_grouped_tiles<MB, DD, OCC, GLU, true, Op><<<a.P, 256, 0, s>>>(a)
           : k_grouped_tiles<MB, DD, OCC, GLU, false, Op><<<a.P, 256, 0, s>>>(a);
}
template <int MB, int DD, class Op>
void launch_op(const GroupedArgs& a, bool glu, hipStream_t s) {
  glu ? launch_tiles<MB, DD, 2, true, Op>(a, s) : launch_tiles<MB, DD, 2, false, Op>(a, s);
}
template <int MB, int DD>
void launch_act(const GroupedArgs& a, bool glu, hipStream_t s) {
  a.cexp ? launch_op<MB, DD, G2F16>(a, glu, s) : launch_op<MB, DD, G2Bf16>(a, glu, s);
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_tune_grouped(int form) {
  if (form < 0 || form > 5) return QW4_ERR_SHAPE;
  g_form.store(form, std::memory_order_relaxed);
  return QW4_OK;
}

int qw4_gemm_grouped(uint16_t* y, const qw4_weights* w, const uint16_t* x, int x_rows,
                     const qw4_plan* plan, int pairs, int gather, const uint16_t* bias, int act,
                     qw4_workspace* ws, void* stream) {
  const int st = check_weights_public(w);
  if (st) return st;
  if (!plan || !plan->offsets) return QW4_ERR_NULL;
  if (plan->experts < 1 || plan->experts > kMaxExperts || w->out_f % plan->experts) return QW4_ERR_SHAPE;
  if (act < QW4_ACT_NONE || act > QW4_ACT_SWIGLU) return QW4_ERR_ACT;
  const bool glu = act == QW4_ACT_SWIGLU;
  const int n = w->out_f / plan->experts;
  if (n % (glu ? 2 * kTileN : kTileN)) return QW4_ERR_SHAPE;
  if (pairs < 0) return QW4_ERR_M;
  if (pairs > plan->max_pairs) return QW4_ERR_SCRATCH;
  if (pairs > 0 && x_rows < (gather ? 1 : pairs)) return QW4_ERR_SHAPE;
  // an expert's weights, and a gathered x, through 32-bit buffer offsets
  const size_t row = (size_t)w->in_f * 2;
  if ((size_t)n * w->in_f / 2 >= (1ull << 32) || (gather && pairs > 0 && (size_t)x_rows * row >= (1ull << 32) - row))
    return QW4_ERR_SHAPE;
  if (pairs == 0) return QW4_OK;
  if (!y || !x || (gather && !plan->tokens)) return QW4_ERR_NULL;
  if (((uintptr_t)y | (uintptr_t)x | (uintptr_t)bias) & 15) return QW4_ERR_ALIGN;
  GroupedArgs a{};
  a.qw = w->qweight;
  a.sc = w->scale;
  a.zr = w->zeros;
  a.x = x;
  a.y = y;
  a.offsets = plan->offsets;
  a.tokens = gather ? plan->tokens : nullptr;
  a.epi = {bias, nullptr, act, glu ? n / 2 : 0};
  a.E = plan->experts;
  a.n = n;
  a.K = w->in_f;
  a.G = w->num_groups;
  a.R = pairs;
  a.x_bytes = gather ? (uint32_t)((size_t)x_rows * row) : 0u;
  a.ld = glu ? n / 2 : n;
  a.tiles_n = (n + G2_BN - 1) / G2_BN;
  const int cus = device_cus();
  const int tuned = g_form.load(std::memory_order_relaxed);
  // The rounding of the weights follows the sizes and the workspace, not what is faster by
  // some microseconds: up to the rows an expert where qw4_linear uses a weight of its size
  // exactly, fp16 operands (11 bits), or without a workspace only the kernels that use it
  // exactly. Beyond, the ungated tiles take bf16 ones as qw4_gemm does: 0.0022 of the output's
  // rms from exact against 0.0017, but without k_half_rows (us, fp16 / bf16: 32 experts, 2176 ->
  // 5120, 125 rows 125 / 116; 64, 1024 -> 2048, 512 rows 182 / 152). Gated, where each factor
  // carries the rounding (0.0027), they take fp16 ones at any size.
  const bool few = (long long)pairs <= (long long)a.E * exact_rows(n, w->in_f);
  const int x_used = gather ? x_rows : pairs;
  const bool half = (glu || (few && tuned != 4)) && ws && ws->buf && ((uintptr_t)ws->buf & 255) == 0 &&
                    ws->bytes >= half_rows_bytes(x_used, w);
  const int form = tuned ? tuned : grouped_form(a, glu, cus, few && !half);
  if (grouped_rows_launch(a, glu, cus, form, (hipStream_t)stream)) {
    QW4_LAUNCH_CHECK();
    return QW4_OK;
  }
  if (half) {
    const HalfRows h = half_rows(ws->buf, x, x_used, w, (hipStream_t)stream);
    a.x = h.x;
    a.rexp = h.rexp;
    a.cexp = h.cexp;
  }
  // 128-row tiles (64-row ones: grouped_form), two workgroups a CU, one's start and end behind
  // the other's products; or 256-row tiles, one a CU, which cost less a row but waste more where
  // an expert ends, hide nothing, and need rounds enough not to idle in the last. us (128 / 256),
  // experts, K -> weight rows, rows an expert: 32, 5120 -> 2048 ungated 768 / 1024 / 1536
  // 511 / 531, 667 / 635, 981 / 915; 64, 2048 -> 4096 512 / 1024 / 1536 583 / 603, 1106 / 1077,
  // 1636 / 1579; gated 64, 2048 -> 2048 768 / 1024 / 1536 488 / 525, 569 / 535, 827 / 782; few
  // rounds: 16, 2048 -> 2048 1024 148 / 163, 64, 2048 -> 1024 768 226 / 253. The gated one has fp16
  // operands only.
  const double tiles8 = (pairs / 256. + 0.5 * a.E) * a.tiles_n;
  const bool high = (long long)pairs >= 900LL * a.E && tiles8 >= 4. * cus && (!glu || a.cexp);
  const int mb = tuned == 4 || (!tuned && high) ? (glu && !a.cexp ? 4 : 8) : form == 5 ? 2 : 4;
  const int occ = mb == 8 ? 1 : 2;
  const long long most = ((long long)pairs / (32 * mb) + std::min(a.E, pairs)) * a.tiles_n;
  if (most > 0x3fffffffLL) return QW4_ERR_SHAPE;
  a.P = (int)std::min<long long>(most, cus * occ);
  hipStream_t s = (hipStream_t)stream;
  if (mb == 8)
    glu ? launch_tiles<8, 2, 1, true, G2F16>(a, s) : launch_tiles<8, 2, 1, false, G2Bf16>(a, s);
  else if (mb == 4)
    launch_act<4, 2>(a, glu, s);
  else
    launch_act<2, 4>(a, glu, s);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // extern "C"
