// Gate for namespace qwen's rows in 8 bits, their products and log probabilities: a norm,
// a gated projection, the one back with the residual and a head as a C++ caller writes
// them, against the formulas in fp64. Exit 0 = pass.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "../../include/qwen_w4a16.hpp"
#include "../../oracle/oracle.h"

#define CK(x)                                                                   \
  do {                                                                          \
    hipError_t e_ = (x);                                                        \
    if (e_ != hipSuccess) {                                                     \
      std::fprintf(stderr, "HIP %s:%d %s\n", __FILE__, __LINE__, hipGetErrorString(e_)); \
      return 2;                                                                 \
    }                                                                           \
  } while (0)

namespace {

std::mt19937 rng(77);
std::normal_distribution<float> normal(0.f, 1.f);

template <class T>
T* upload(const std::vector<T>& h) {
  T* d = nullptr;
  if (hipMalloc(&d, h.size() * sizeof(T)) != hipSuccess ||
      hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess)
    std::exit(2);
  return d;
}
__hip_bfloat16* bf(uint16_t* p) { return reinterpret_cast<__hip_bfloat16*>(p); }

std::vector<uint16_t> random_bf16(size_t n, float scale) {
  std::vector<uint16_t> v(n);
  for (auto& x : v) x = or_f32_to_bf16(normal(rng) * scale);
  return v;
}

// Random weights [N][K], repacked, and their values.
qwen::W4A16Weights random_weights(int N, int K, std::vector<double>& values) {
  const int G = K / 128;
  std::vector<uint8_t> q((size_t)N * K), zp((size_t)N * G);
  std::vector<uint16_t> s((size_t)N * G), scale((size_t)N * G);
  for (auto& v : q) v = rng() & 15;
  for (auto& v : zp) v = rng() & 15;
  for (auto& v : s) v = or_f32_to_bf16(std::fabs(normal(rng) * 0.02f) + 1e-4f);
  std::vector<uint32_t> packed((size_t)N * K / 8), zpw((size_t)N / 8 * G);
  or_pack_ct(q.data(), zp.data(), s.data(), N, K, 128, packed.data(), scale.data(), zpw.data());
  values.resize((size_t)N * K);
  for (int n = 0; n < N; ++n)
    for (int k = 0; k < K; ++k)
      values[(size_t)n * K + k] =
          ((int)q[(size_t)n * K + k] - (int)zp[(size_t)n * G + k / 128]) * (double)or_bf16_to_f32(s[(size_t)n * G + k / 128]);
  uint32_t *dp = upload(packed), *dz = upload(zpw);
  uint16_t* ds = upload(scale);
  qwen::W4A16Weights w;
  qwen::awq_repack(w, dp, bf(ds), dz, N, K, 128);
  if (hipDeviceSynchronize() != hipSuccess) std::exit(2);
  (void)hipFree(dp);
  (void)hipFree(ds);
  (void)hipFree(dz);
  return w;
}

double dot(const double* w, const double* x, int K) {
  double v = 0;
  for (int k = 0; k < K; ++k) v += w[k] * x[k];
  return v;
}
double silu(double v) { return v / (1 + std::exp(-v)); }


std::vector<double> rows_of(const uint16_t* d, size_t n) {
  std::vector<uint16_t> h(n);
  if (hipMemcpy(h.data(), d, n * 2, hipMemcpyDeviceToHost) != hipSuccess) std::exit(2);
  std::vector<double> v(n);
  for (size_t i = 0; i < n; ++i) v[i] = or_bf16_to_f32(h[i]);
  return v;
}

// Largest difference over the largest value.
bool near(const char* what, const std::vector<double>& ref, const std::vector<double>& got, double bound) {
  double most = 0, off = 0;
  for (size_t i = 0; i < ref.size(); ++i) {
    most = std::max(most, std::fabs(ref[i]));
    off = std::max(off, std::fabs(ref[i] - got[i]));
  }
  std::printf("%s: %.6f (bound %.6f)\n", what, off / most, bound);
  return off <= bound * most;
}

}  // namespace

int main() {
  const int H = 384, I = 256, V = 1088, k = 5, most = 150;
  std::vector<double> gu, dn, hd;
  qwen::W4A16Weights wu = random_weights(2 * I, H, gu), wd = random_weights(H, I, dn), wh = random_weights(V, H, hd);
  const std::vector<uint16_t> nw = random_bf16(H, 0.1f);
  uint16_t* dw = upload(nw);
  qw4_a8 a, b;
  qwen::a8_alloc(a, most, H);
  qwen::a8_alloc(b, most, I);
  qwen::GemmWorkspace ws;
  qwen::gemm_workspace_alloc(ws, 128u << 20);
  hipStream_t stream;
  CK(hipStreamCreate(&stream));
  bool ok = true;
  for (int T : {1, 9, 40, most}) {
    const std::vector<uint16_t> h0 = random_bf16((size_t)T * H, 1.f), r0 = random_bf16((size_t)T * H, 1.f);
    uint16_t *h = upload(h0), *r = upload(r0), *mid = upload(std::vector<uint16_t>((size_t)T * I));
    uint16_t *va = upload(std::vector<uint16_t>((size_t)T * H)), *vb = upload(std::vector<uint16_t>((size_t)T * I));
    float* logits = upload(std::vector<float>((size_t)T * V));
    std::vector<int32_t> asked(2 * T);
    for (int i = 0; i < 2 * T; ++i) asked[i] = (int)(rng() % (V + 1));   // V: outside
    int32_t *dt = upload(asked), *ids = upload(std::vector<int32_t>((size_t)T * k));
    float *lp = upload(std::vector<float>(2 * T)), *ent = upload(std::vector<float>(T)), *top = upload(std::vector<float>((size_t)T * k));
    qwen::rmsnorm_a8(a, bf(h), bf(h), bf(r), bf(dw), T, 1e-6f, stream);
    qwen::a8_dequant_rows(bf(va), a, 0, T, stream);
    qwen::linear_w4a8(bf(mid), wu, a, T, nullptr, QW4_ACT_SWIGLU, nullptr, ws, stream);
    qwen::quantize_a8(b, bf(mid), I, T, stream);
    qwen::a8_dequant_rows(bf(vb), b, 0, T, stream);
    qwen::linear_w4a8(bf(h), wd, b, T, nullptr, QW4_ACT_NONE, bf(h), ws, stream);
    CK(hipStreamSynchronize(stream));
    // every step from what the one before has stored
    std::vector<double> sum((size_t)T * H), norm((size_t)T * H), m((size_t)T * I), out((size_t)T * H);
    const std::vector<double> qa = rows_of(va, norm.size()), got_m = rows_of(mid, m.size()), qb = rows_of(vb, m.size());
    for (int t = 0; t < T; ++t) {
      double ss = 0;
      for (int i = 0; i < H; ++i) {
        const size_t at = (size_t)t * H + i;
        sum[at] = or_bf16_to_f32(or_f32_to_bf16(or_bf16_to_f32(h0[at]) + or_bf16_to_f32(r0[at])));
        ss += sum[at] * sum[at];
      }
      for (int i = 0; i < H; ++i)
        norm[(size_t)t * H + i] = sum[(size_t)t * H + i] / std::sqrt(ss / H + 1e-6) * (1 + or_bf16_to_f32(nw[i]));
      const double* x = &qa[(size_t)t * H];
      for (int i = 0; i < I; ++i)
        m[(size_t)t * I + i] = silu(dot(&gu[(size_t)i * H], x, H)) * dot(&gu[(size_t)(I + i) * H], x, H);
      for (int c = 0; c < H; ++c)
        out[(size_t)t * H + c] = dot(&dn[(size_t)c * I], &qb[(size_t)t * I], I) + sum[(size_t)t * H + c];
    }
    // half a step of 1/127 of the group's largest value, and the bf16 that is read back
    ok = near("norm in 8 bits", norm, qa, 0.5 / 127 + 0x1p-8) && ok;
    ok = near("rows in 8 bits", got_m, qb, 0.5 / 127 + 0x1p-8) && ok;
    // both factors' and the result's roundings to bf16: values read back and stored
    ok = near("gated projection", m, got_m, 0.015) && ok;
    ok = near("projection and residual", out, rows_of(h, out.size()), 0.01) && ok;

    qwen::quantize_a8(a, bf(h), H, T, stream);
    qwen::a8_dequant_rows(bf(va), a, 0, T, stream);
    qwen::linear_w4a8_f32(logits, wh, a, T, ws, stream);
    qwen::logprobs_f32(lp, ent, ids, top, logits, V, dt, T, V, 2, k, ws, stream);
    CK(hipStreamSynchronize(stream));
    std::vector<float> lg((size_t)T * V), glp(2 * T), gent(T), gtop((size_t)T * k);
    std::vector<int32_t> gid((size_t)T * k);
    CK(hipMemcpy(lg.data(), logits, lg.size() * 4, hipMemcpyDeviceToHost));
    CK(hipMemcpy(glp.data(), lp, glp.size() * 4, hipMemcpyDeviceToHost));
    CK(hipMemcpy(gent.data(), ent, gent.size() * 4, hipMemcpyDeviceToHost));
    CK(hipMemcpy(gtop.data(), top, gtop.size() * 4, hipMemcpyDeviceToHost));
    CK(hipMemcpy(gid.data(), ids, gid.size() * 4, hipMemcpyDeviceToHost));
    const std::vector<double> qh = rows_of(va, (size_t)T * H);
    std::vector<double> want((size_t)T * V), got(lg.begin(), lg.end());
    double off = 0;
    for (int t = 0; t < T; ++t) {
      for (int n = 0; n < V; ++n) want[(size_t)t * V + n] = dot(&hd[(size_t)n * H], &qh[(size_t)t * H], H);
      const float* x = &lg[(size_t)t * V];
      double L = 0, mx = -1e30, mn = 1e30, e = 0;
      for (int n = 0; n < V; ++n) {
        mx = std::max(mx, (double)x[n]);
        mn = std::min(mn, (double)x[n]);
      }
      for (int n = 0; n < V; ++n) L += std::exp(x[n] - mx);
      L = mx + std::log(L);
      for (int n = 0; n < V; ++n) e -= std::exp(x[n] - L) * (x[n] - L);
      // x - m and (x - m) - log: half a step of at most mx - mn, and of that and log V, the log
      // (at most log V = 7) a few steps: 2^-24 (2 (mx - mn) + 64) in all, up to 2e-4 here, where
      // logits differ by some hundreds. The entropy has factors exp(x - m) on x - m, which keep
      // its terms below log V: 64 steps of 2^-24.
      const double step = 0x1p-24 * (2 * (mx - mn) + 64);
      off = std::max(off, std::fabs(e - gent[t]) / (64 * 0x1p-24 * (1 + std::log((double)V))));
      for (int j = 0; j < 2; ++j) {
        const int id = asked[2 * t + j];
        off = std::max(off, std::fabs((id < V ? x[id] - L : 0) - glp[2 * t + j]) / step);
      }
      std::vector<char> used(V, 0);
      for (int j = 0; j < k; ++j) {
        int best = -1;
        for (int n = 0; n < V; ++n)
          if (!used[n] && (best < 0 || x[n] > x[best])) best = n;
        used[best] = 1;
        ok = gid[(size_t)t * k + j] == best && ok;
        off = std::max(off, std::fabs(x[best] - L - gtop[(size_t)t * k + j]) / step);
      }
    }
    ok = near("logits", want, got, 0x1p-8) && ok;   // the values read back in bf16
    std::printf("log probabilities: %.2f of their bound\n", off);
    ok = off < 1 && ok;
    for (void* p : {(void*)h, (void*)r, (void*)mid, (void*)va, (void*)vb, (void*)logits, (void*)dt, (void*)ids, (void*)lp, (void*)ent, (void*)top})
      CK(hipFree(p));
  }
  qwen::a8_free(a);
  qwen::a8_free(b);
  qwen::gemm_workspace_free(ws);
  for (qwen::W4A16Weights* w : {&wu, &wd, &wh}) qwen::awq_free(*w);
  CK(hipFree(dw));
  CK(hipStreamDestroy(stream));
  std::printf(ok ? "gate_a8: PASS\n" : "gate_a8: FAIL\n");
  return ok ? 0 : 1;
}
