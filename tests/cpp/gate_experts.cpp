// Gate for namespace qwen's layers of experts and products with an epilogue: a layer of
// experts as a C++ caller writes it, and a projection with bias, activation and residual,
// against the formulas in fp64. Exit 0 = pass.
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

// Largest difference over the largest value: the products' and hidden values' roundings
// to bf16 are 2^-8 each of values below the largest.
bool near(const char* what, const std::vector<double>& ref, uint16_t* d, double bound) {
  std::vector<uint16_t> got(ref.size());
  if (hipMemcpy(got.data(), d, got.size() * 2, hipMemcpyDeviceToHost) != hipSuccess) std::exit(2);
  double most = 0, off = 0;
  for (size_t i = 0; i < ref.size(); ++i) {
    most = std::max(most, std::fabs(ref[i]));
    off = std::max(off, std::fabs(ref[i] - or_bf16_to_f32(got[i])));
  }
  std::printf("%s: %.5f (bound %.5f)\n", what, off / most, bound);
  return off <= bound * most;
}

}  // namespace

int main() {
  const int T = 9, E = 4, k = 2, H = 256, I = 128;
  std::vector<double> gu, dn;
  qwen::W4A16Weights wu = random_weights(E * 2 * I, H, gu), wd = random_weights(E * H, I, dn);
  const std::vector<uint16_t> x = random_bf16((size_t)T * H, 1.f), res = random_bf16((size_t)T * H, 1.f);
  std::vector<uint16_t> logits = random_bf16((size_t)T * E, 1.f);
  for (int e = 0; e < E; ++e) logits[(size_t)(T - 1) * E + e] = 0xff80;   // -Inf: a padding row
  uint16_t *dx = upload(x), *dl = upload(logits), *dr = upload(res);
  uint16_t *h = upload(std::vector<uint16_t>((size_t)T * k * I)), *y = upload(std::vector<uint16_t>((size_t)T * k * H));
  int32_t* ids = upload(std::vector<int32_t>((size_t)T * k));
  float* wt = upload(std::vector<float>((size_t)T * k));
  qw4_plan plan;
  qwen::expert_plan_alloc(plan, E, T * k);
  qwen::GemmWorkspace ws;
  qwen::gemm_workspace_alloc(ws, qwen::epilogue_workspace(wu, T));
  hipStream_t stream;
  CK(hipStreamCreate(&stream));
  auto products = [&] {
    qwen::gemm_grouped_w4a16(bf(h), wu, bf(dx), T, plan, T * k, true, nullptr, QW4_ACT_SWIGLU, ws, stream);
    qwen::gemm_grouped_w4a16(bf(y), wd, bf(h), T * k, plan, T * k, false, nullptr, QW4_ACT_NONE, ws, stream);
    qwen::combine_experts(bf(dr), bf(y), plan, wt, T, k, H, bf(dr), stream);   // into the residual
  };
  qwen::route_experts(ids, wt, &plan, bf(dl), T, E, k, true, stream);
  products();
  CK(hipStreamSynchronize(stream));

  std::vector<double> xd((size_t)T * H), ref((size_t)T * H);
  for (size_t i = 0; i < xd.size(); ++i) xd[i] = or_bf16_to_f32(x[i]);
  for (int t = 0; t < T; ++t) {
    double* out = &ref[(size_t)t * H];
    for (int j = 0; j < H; ++j) out[j] = or_bf16_to_f32(res[(size_t)t * H + j]);
    if (t == T - 1) continue;   // no expert
    int best[2] = {-1, -1};
    double v[2] = {0, 0};
    for (int j = 0; j < k; ++j)
      for (int e = 0; e < E; ++e) {
        const double l = or_bf16_to_f32(logits[(size_t)t * E + e]);
        if (!(j && e == best[0]) && (best[j] < 0 || l > v[j])) {
          best[j] = e;
          v[j] = l;
        }
      }
    const double m1 = std::exp(v[1] - v[0]);
    for (int j = 0; j < k; ++j) {
      const int e = best[j];
      double hid[I];
      for (int i = 0; i < I; ++i)
        hid[i] = silu(dot(&gu[((size_t)e * 2 * I + i) * H], &xd[(size_t)t * H], H)) *
                 dot(&gu[((size_t)e * 2 * I + I + i) * H], &xd[(size_t)t * H], H);
      for (int c = 0; c < H; ++c)
        out[c] += (j ? m1 : 1.) / (1 + m1) * dot(&dn[((size_t)e * H + c) * I], hid, I);
    }
  }
  bool ok = near("layer of experts", ref, dr, 0.02);
  // the same plan from the ids, and fp32 logits
  std::vector<float> lf(logits.size());
  for (size_t i = 0; i < lf.size(); ++i) lf[i] = or_bf16_to_f32(logits[i]);
  float* dlf = upload(lf);
  CK(hipMemcpy(dr, res.data(), res.size() * 2, hipMemcpyHostToDevice));
  qwen::route_experts_f32(ids, wt, nullptr, dlf, T, E, k, true, stream);
  qwen::route_expert_ids(plan, ids, T, k, stream);
  products();
  CK(hipStreamSynchronize(stream));
  ok = near("plan from ids", ref, dr, 0.02) && ok;

  // a projection with bias, activation and residual in y: decode rows and prefill tiles
  qwen::GemvScratch scratch;
  qwen::gemv_scratch_alloc(scratch, H, E * 2 * I, 128, 16);
  for (int rows : {1, 9, 150}) {
    const int N = E * 2 * I;
    const std::vector<uint16_t> xr = random_bf16((size_t)rows * H, 1.f), b = random_bf16(N, 1.f),
                                r0 = random_bf16((size_t)rows * N, 1.f);
    uint16_t *dxr = upload(xr), *db = upload(b), *dy = upload(r0);
    qwen::linear_epilogue_w4a16(bf(dy), wu, bf(dxr), rows, bf(db), QW4_ACT_GELU, bf(dy), scratch, ws, stream);
    CK(hipStreamSynchronize(stream));
    std::vector<double> xf(xr.size()), want((size_t)rows * N);
    for (size_t i = 0; i < xf.size(); ++i) xf[i] = or_bf16_to_f32(xr[i]);
    for (int t = 0; t < rows; ++t)
      for (int n = 0; n < N; ++n) {
        const double v = dot(&gu[(size_t)n * H], &xf[(size_t)t * H], H) + or_bf16_to_f32(b[n]);
        want[(size_t)t * N + n] = 0.5 * v * std::erfc(-v / std::sqrt(2.)) + or_bf16_to_f32(r0[(size_t)t * N + n]);
      }
    ok = near("projection with an epilogue", want, dy, 0.01) && ok;
    CK(hipFree(dxr));
    CK(hipFree(db));
    CK(hipFree(dy));
  }
  qwen::expert_plan_free(plan);
  qwen::gemm_workspace_free(ws);
  qwen::gemv_scratch_free(scratch);
  qwen::awq_free(wu);
  qwen::awq_free(wd);
  std::printf(ok ? "gate_experts: PASS\n" : "gate_experts: FAIL\n");
  return ok ? 0 : 1;
}
