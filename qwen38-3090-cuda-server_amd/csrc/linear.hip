// The reference's linear() path choice (src/model/model.cu:522-565,
// :643-658) over this library's kernels: the GEMV for one row, the skinny
// kernel in chunks of 16 or 32 rows while it reads the weights fewer times
// than the prefill GEMM would cost, the prefill GEMM beyond. Host code only.
#include <atomic>

#include "../../include/qwen_w4a16.h"
#include "epilogue.h"
#include "skinny.h"

namespace qw4 {
int check_weights_public(const qw4_weights* w);
}

namespace {

std::atomic<int> g_lin_max_t{0};   // qw4_tune_linear override (0: the rule below)

int lin_max_t(const qw4_weights* w) {
  const int v = g_lin_max_t.load(std::memory_order_relaxed);
  return v > 0 ? v : qw4::exact_rows(w->out_f, w->in_f);
}

// T rows of y [T][width] in skinny passes, with the epilogue e or without (null).
int few_rows(uint16_t* y, int width, const qw4_weights* w, const uint16_t* x, int T, qw4_scratch* s,
             const qw4::Epilogue* e, void* stream) {
  const int chunk = s->max_m < 16 ? s->max_m : 16;
  if (chunk < 1) return QW4_ERR_SCRATCH;
  for (int i = 0, n; i < T; i += n) {
    uint16_t* const yi = y + (size_t)i * width;
    const uint16_t* const xi = x + (size_t)i * w->in_f;
    qw4::Epilogue ei{};
    if (e) {
      ei = *e;
      if (ei.res) ei.res += (size_t)i * width;
    }
    // two 16-row passes in one where it pays; in qw4_linear a last single row stays
    // a pass of its own (the GEMV's sums)
    const int left = T - i;
    n = left < 32 ? left : 32;
    if (!e && n % 16 == 1) --n;
    if (chunk == 16 && n > 16) {
      bool taken = false;
      const int st = qw4::skinny_rows32(yi, w, xi, n, s, stream, e ? &ei : nullptr, &taken);
      if (st) return st;
      if (taken) continue;
    }
    n = left < chunk ? left : chunk;
    const int st = e ? qw4::skinny_epilogue(yi, w, xi, n, s, ei, stream)
                     : qw4_gemm_small(yi, w, xi, n, s, stream);
    if (st) return st;
  }
  return QW4_OK;
}

}  // namespace

// Rows up to which skinny passes run instead of the prefill GEMM: they use the
// weights exactly where the GEMM rounds them to bf16, so this line is not moved
// with every change of either's speed. 16 whole passes under the ratio that
// 16-row passes (0.245 us per MB of weights + 5.8 us) and the GEMM (60 us + 0.4
// us per MB) had on MI355X when it was set: 48 rows for gate|up (93 MB), 64 for
// down (46 MB), 96 for qkv (19 MB), 112 for o_proj (11 MB).
int qw4::exact_rows(int out_f, int in_f) {
  const double mb = (double)out_f * in_f * (0.5 + 2.5 / 128) / 1e6;
  const int chunks = (int)((60.0 + 0.4 * mb) / (0.245 * mb + 5.8));
  return 16 * (chunks < 1 ? 1 : chunks);
}

extern "C" {

int qw4_tune_linear(int max_t) {
  if (max_t < 0) return QW4_ERR_SHAPE;
  g_lin_max_t.store(max_t, std::memory_order_relaxed);
  return 0;
}

int qw4_linear_max_t(const qw4_weights* w) {
  if (!w || w->out_f <= 0 || w->in_f <= 0) return QW4_ERR_NULL;
  return lin_max_t(w);
}

int qw4_linear(uint16_t* y, const qw4_weights* w, const uint16_t* x, int T, qw4_scratch* s,
               qw4_workspace* ws, void* stream) {
  if (!y || !w || !x) return QW4_ERR_NULL;
  if (T < 1) return QW4_ERR_M;
  if (T == 1) return qw4_gemv(y, w, x, s, stream);
  if (T <= lin_max_t(w) && s) return few_rows(y, w->out_f, w, x, T, s, nullptr, stream);
  return qw4_gemm(y, w, x, T, ws, stream);
}

int qw4_linear_epilogue(uint16_t* y, const qw4_weights* w, const uint16_t* x, int T,
                        const uint16_t* bias, int act, const uint16_t* residual, qw4_scratch* s,
                        qw4_workspace* ws, void* stream) {
  const int st = qw4::check_weights_public(w);
  if (st) return st;
  if (!y || !x) return QW4_ERR_NULL;
  if (T < 1) return QW4_ERR_M;
  if (act < QW4_ACT_NONE || act > QW4_ACT_SWIGLU) return QW4_ERR_ACT;
  if (act == QW4_ACT_SWIGLU && w->out_f % (2 * qw4::kTileN)) return QW4_ERR_SHAPE;
  if (((uintptr_t)y | (uintptr_t)x | (uintptr_t)bias | (uintptr_t)residual) & 15) return QW4_ERR_ALIGN;
  const qw4::Epilogue e{bias, residual, act, act == QW4_ACT_SWIGLU ? w->out_f / 2 : 0};
  if (s && T <= lin_max_t(w)) return few_rows(y, w->out_f - e.up, w, x, T, s, &e, stream);
  return qw4::gemm_epilogue(y, w, x, T, ws, e, stream);
}

}  // extern "C"
