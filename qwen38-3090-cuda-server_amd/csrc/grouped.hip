// W4A16 products grouped by expert: rows [offsets[e], offsets[e + 1]) of y are f(x_row
// W_e^T + b_e), the experts' weights stacked in one W4A16 tensor, x in the plan's order
// or gathered by its tokens. The row counts live on the device only: every workgroup
// reads the offsets and finds its own work, so that no call waits for the host and a
// captured graph routes anew on every replay.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/qwen_w4a16.h"
#include "gemm_tile.h"
#include "grouped.h"
#include "skinny.h"
#include "w4a16_common.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);

namespace {

// Many rows an expert: the MFMA tile of the prefill GEMM (gemm_tile.h) over (expert, row
// block, column tile). Tiles go expert by expert, a column tile's row blocks together,
// and an XCD takes a run of them: its weights and rows stay in its L2. Every workgroup
// takes every P-th tile.
template <int MB, bool GLU, bool GATHER>
__global__ __launch_bounds__(256, 1) void k_grouped_tiles(GroupedArgs a) {
  using Sp = G2Split<2, 4, MB>;
  __shared__ u32x4 lds[Sp::DEPTH][32 * MB * 16];
  __shared__ int start[kMaxExperts + 1];
  __shared__ int wsum[4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int all = __builtin_amdgcn_readfirstlane(block_starts<32 * MB, 256>(a, start, wsum)) * a.tiles_n;
  const uint32_t row_bytes = (uint32_t)a.K * 2u;
  const int srow = 4 * wave + (lane >> 4);   // row within the 16-row swizzle period
  const uint32_t chunk = (uint32_t)((lane & 15) ^ srow) * 16u;
  const int up = a.epi.up / kTileN;
  const int width = GLU ? a.ld : a.n;   // columns the column tiles run over
  f32x16v acc[2][MB];
  for (int t = a.P % 8 ? (int)blockIdx.x : (int)((blockIdx.x & 7) * (a.P >> 3) + (blockIdx.x >> 3)); t < all;
       t += a.P) {
    const int e = expert_of(start, a.E, a.tiles_n, t);
    int lo, hi;
    expert_rows(a, e, lo, hi);
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int blocks = max(1, (hi - lo + 32 * MB - 1) / (32 * MB));
    const int at = t - __builtin_amdgcn_readfirstlane(start[e]) * a.tiles_n;
    if ((uint32_t)at >= (uint32_t)(blocks * a.tiles_n)) continue;   // offsets of no plan
    const int tn = at / blocks, m0 = lo + (at - tn * blocks) * 32 * MB;
    const int rows = hi - m0;
    // a wave's weight tile, half and first output column, as the dense product's
    const int wt = GLU ? tn * 2 + (wave >> 1) : tn * 4 + wave;
    const int b0 = GLU ? wave & 1 : 0;
    const int col = wt * kTileN + 32 * b0;
    const bool valid = wt * kTileN < width;
    const int ltile = valid ? wt : width / kTileN - 1;
    const size_t blk = (size_t)e * (a.n / kTileN) * a.G;   // the expert's first weight block
    const G2Rsrc wr = g2_weights(a.qw + blk * kWordsPerBlock, a.sc + blk * kMetaU16, a.zr + blk * 16, a.n, a.G);
    const G2Rsrc none =
        g2_weights(a.qw + blk * kWordsPerBlock, a.sc + blk * kMetaU16, a.zr + blk * 16, a.n, a.G, false);
    if constexpr (GATHER) {
      G2Gather<Sp::ACT> from;
#pragma unroll
      for (int i = 0; i < Sp::ACT; ++i) {
        const int r = 4 * (4 * i + wave) + (lane >> 4);
        const int row = r < rows ? a.tokens[m0 + r] : -1;
        const uint64_t off = (uint64_t)(uint32_t)row * row_bytes;   // past x: reads as zeros
        from.off[i] = off < a.x_bytes ? (uint32_t)off + chunk : a.x_bytes;
      }
      g2_segment<2, 4, MB, GLU>(a.G, wr, none, g2_rsrc(a.x, a.x_bytes), g2_rsrc(a.x, 0), from, lds, acc,
                                ltile, up, b0, 0, 0, a.G, wave, lane);
    } else {
      const uint16_t* x0 = a.x + (size_t)m0 * a.K;
      const G2Rows from{(uint32_t)(lane >> 4) * row_bytes + chunk, row_bytes};
      g2_segment<2, 4, MB, GLU>(a.G, wr, none, g2_rsrc(x0, (uint32_t)min(rows, 32 * MB) * row_bytes),
                                g2_rsrc(x0, 0), from, lds, acc, ltile, up, b0, 0, 0, a.G, wave, lane);
    }
    Epilogue ep = a.epi;
    if (ep.bias) ep.bias += (size_t)e * a.n + col;
    g2_store_epilogue<MB, GLU>(acc, &lds[0][0], a.y + (size_t)m0 * a.ld + col, ep, a.ld, rows, valid, wave,
                               lane);
  }
}

int device_cus() {
  static std::atomic<int> cus[kMaxDevices];
  std::atomic<int>& v = cus[current_device()];
  int n = v.load(std::memory_order_relaxed);
  if (!n) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
    v.store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int MB>
void launch_tiles(const GroupedArgs& a, bool glu, hipStream_t s) {
  if (glu)
    a.tokens ? k_grouped_tiles<MB, true, true><<<a.P, 256, 0, s>>>(a)
             : k_grouped_tiles<MB, true, false><<<a.P, 256, 0, s>>>(a);
  else
    a.tokens ? k_grouped_tiles<MB, false, true><<<a.P, 256, 0, s>>>(a)
             : k_grouped_tiles<MB, false, false><<<a.P, 256, 0, s>>>(a);
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_gemm_grouped(uint16_t* y, const qw4_weights* w, const uint16_t* x, int x_rows,
                     const qw4_plan* plan, int pairs, int gather, const uint16_t* bias, int act,
                     qw4_workspace* ws, void* stream) {
  (void)ws;
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
  if (x_rows < 0 || (!gather && x_rows < pairs)) return QW4_ERR_SHAPE;
  // an expert's weights, and a gathered x, through 32-bit buffer offsets
  const size_t row = (size_t)w->in_f * 2;
  if ((size_t)n * w->in_f / 2 >= (1ull << 32) || (gather && (size_t)x_rows * row >= (1ull << 32) - row))
    return QW4_ERR_SHAPE;
  if (pairs == 0 || x_rows == 0) return QW4_OK;
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
  if (grouped_rows_launch(a, glu, cus, (hipStream_t)stream)) {
    QW4_LAUNCH_CHECK();
    return QW4_OK;
  }
  constexpr int mb = 4;
  const long long most = ((long long)pairs / (32 * mb) + std::min(a.E, pairs)) * a.tiles_n;
  if (most > 0x7fffffffLL) return QW4_ERR_SHAPE;
  a.P = (int)std::min<long long>(most, cus);
  launch_tiles<mb>(a, glu, (hipStream_t)stream);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // extern "C"
