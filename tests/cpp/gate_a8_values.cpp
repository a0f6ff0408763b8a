// Gate for namespace qwen's rows in 8 bits, their products and log probabilities, value by
// value: every one has to be within its own bound of the formula in fp64, which NaN is not.
// Exit 0 = pass.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <limits>
#include <random>
#include <vector>

#include "../../include/qwen_w4a16.hpp"
#include "../../oracle/oracle.h"

#define CK(x)                                                                   \
  do {                                                                          \
    hipError_t e_ = (x);                                                        \
    if (e_ != hipSuccess) {                                                     \
      std::fprintf(stderr, "HIP %s:%d %s\n", __FILE__, __LINE__, hipGetErrorString(e_)); \
      std::exit(2);                                                             \
    }                                                                           \
  } while (0)

namespace {

std::mt19937 rng(5);
std::normal_distribution<float> normal(0.f, 1.f);

template <class T>
struct Device {
  T* p = nullptr;
  size_t n;
  explicit Device(const std::vector<T>& h) : n(h.size()) {
    CK(hipMalloc(&p, n * sizeof(T)));
    CK(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice));
  }
  Device(size_t n, int byte) : n(n) {   // every byte the same: 0xff is NaN in bf16 and fp32
    CK(hipMalloc(&p, n * sizeof(T)));
    CK(hipMemset(p, byte, n * sizeof(T)));
  }
  ~Device() { (void)hipFree(p); }
  Device(const Device&) = delete;
  std::vector<T> host() const {
    std::vector<T> h(n);
    CK(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
    return h;
  }
};
__hip_bfloat16* bf(const Device<uint16_t>& d) { return reinterpret_cast<__hip_bfloat16*>(d.p); }
std::vector<double> doubles(const Device<uint16_t>& d) {
  std::vector<double> v;
  for (uint16_t b : d.host()) v.push_back(or_bf16_to_f32(b));
  return v;
}
std::vector<uint16_t> random_bf16(size_t n, float scale) {
  std::vector<uint16_t> v(n);
  for (auto& x : v) x = or_f32_to_bf16(normal(rng) * scale);
  return v;
}

// Values of one kind, checked one by one.
struct Check {
  const char* what;
  size_t bad = 0, seen = 0;
  void operator()(double got, double want, double bound) {
    ++seen;
    if (!(std::fabs(got - want) <= bound)) ++bad;
  }
  bool ok() const {
    std::printf("%s: %zu of %zu values out of their bounds\n", what, bad, seen);
    return bad == 0 && seen > 0;
  }
};

// Random weights [N][K], repacked, and their values.
qwen::W4A16Weights random_weights(int N, int K, std::vector<double>& values) {
  const int G = K / 128;
  std::vector<uint8_t> q((size_t)N * K), zp((size_t)N * G);
  std::vector<uint16_t> s((size_t)N * G), scale((size_t)N * G);
  for (auto& v : q) v = rng() & 15;
  for (auto& v : zp) v = rng() & 15;
  for (auto& v : s) v = or_f32_to_bf16(0.01f + 0.02f * (rng() % 1000) / 1000.f);
  std::vector<uint32_t> packed((size_t)N * K / 8), zpw((size_t)N / 8 * G);
  or_pack_ct(q.data(), zp.data(), s.data(), N, K, 128, packed.data(), scale.data(), zpw.data());
  values.resize((size_t)N * K);
  for (int n = 0; n < N; ++n)
    for (int k = 0; k < K; ++k)
      values[(size_t)n * K + k] =
          ((int)q[(size_t)n * K + k] - (int)zp[(size_t)n * G + k / 128]) * (double)or_bf16_to_f32(s[(size_t)n * G + k / 128]);
  Device<uint32_t> dp(packed), dz(zpw);
  Device<uint16_t> ds(scale);
  qwen::W4A16Weights w;
  qwen::awq_repack(w, dp.p, bf(ds), dz.p, N, K, 128);
  CK(hipDeviceSynchronize());
  return w;
}

// The values that rows in 8 bits hold, from the arrays themselves.
std::vector<double> held(const qw4_a8& a, int T) {
  const int K = a.in_f;
  std::vector<int8_t> q((size_t)T * K);
  std::vector<float> s((size_t)K / 128 * a.max_rows);
  CK(hipMemcpy(q.data(), a.q, q.size(), hipMemcpyDeviceToHost));
  CK(hipMemcpy(s.data(), a.scale, s.size() * 4, hipMemcpyDeviceToHost));
  // input 8 w + e of a chunk of 32 at byte 4 w + low[e], or 16 + 4 w + high[e]
  static const int low[8] = {0, 2, -1, -1, 1, 3, -1, -1}, high[8] = {-1, -1, 0, 2, -1, -1, 1, 3};
  std::vector<double> v((size_t)T * K);
  for (int t = 0; t < T; ++t)
    for (int i = 0; i < K; ++i) {
      const int w = i % 32 / 8, e = i % 8, at = i / 32 * 32 + 4 * w + (low[e] >= 0 ? low[e] : 16 + high[e]);
      v[(size_t)t * K + i] = q[(size_t)t * K + at] * (double)s[(size_t)(i / 128) * a.max_rows + t];
    }
  return v;
}
// Row t against weight n: the sum, and that of its terms' magnitudes by group.
double dot(const std::vector<double>& w, const std::vector<double>& x, int n, int t, int K, double& size) {
  double v = 0;
  size = 0;
  for (int g = 0; g < K; g += 128) {
    double part = 0;
    for (int k = g; k < g + 128; ++k) part += w[(size_t)n * K + k] * x[(size_t)t * K + k];
    v += part;
    size += std::fabs(part);
  }
  return v;
}
// fp32 sums: two roundings a group, some at the end.
double sum_bound(double size, int K) { return (2 * K / 128 + 8) * 0x1p-24 * size; }

// Every value of rows in 8 bits: half a step of its group's, and the values' own error.
void codes(Check& c, const std::vector<double>& want, const std::vector<double>& got, double rel) {
  for (size_t g = 0; g < want.size(); g += 128) {
    double top = 0;
    for (size_t i = g; i < g + 128; ++i) top = std::max(top, std::fabs(want[i]));
    for (size_t i = g; i < g + 128; ++i) c(got[i], want[i], (0.5 + 127 * 8 * 0x1p-24) * top / 127 + rel * top);
  }
}

}  // namespace

int main() {
  {   // the check itself
    Check c{"planted"};
    c(1.0, 1.0, 0.0);
    c(std::nan(""), 1.0, 1e9);
    c(1.0, std::nan(""), 1e9);
    c(std::numeric_limits<double>::infinity(), 1.0, 1e9);
    if (c.bad != 3) return 1;
  }
  const int H = 384, I = 256, V = 1088, k = 5, asked = 2, most = 130;
  std::vector<double> up, down, head;
  qwen::W4A16Weights wu = random_weights(2 * I, H, up), wd = random_weights(H, I, down), wh = random_weights(V, H, head);
  const std::vector<uint16_t> norm_w = random_bf16(H, 0.1f);
  Device<uint16_t> nw(norm_w);
  qw4_a8 a, b;
  qwen::a8_alloc(a, most, H);
  qwen::a8_alloc(b, most, I);
  qwen::GemmWorkspace ws;
  qwen::gemm_workspace_alloc(ws, 128u << 20);
  Check cn{"norm in 8 bits"}, cu{"gated projection"}, cq{"rows in 8 bits"}, cd{"projection and residual"}, cb{"rows read back"},
      cl{"logits"}, cp{"log probabilities"}, ce{"entropy"}, ct{"alternatives"}, ci{"their ids"};
  for (int T : {1, 12, 40, most}) {
    const std::vector<uint16_t> h0 = random_bf16((size_t)T * H, 1.f), r0 = random_bf16((size_t)T * H, 1.f);
    std::vector<int32_t> ask((size_t)T * asked);
    for (auto& i : ask) i = (int)(rng() % (V + 1));   // V: outside
    Device<uint16_t> h(h0), r(r0), mid((size_t)T * I, 0xff), back((size_t)T * I, 0xff), out((size_t)T * H, 0xff);
    Device<float> logits((size_t)T * V, 0xff), lp((size_t)T * asked, 0xff), ent((size_t)T, 0xff), top((size_t)T * k, 0xff);
    Device<int32_t> ids((size_t)T * k, 0xff), targets(ask);
    qwen::rmsnorm_a8(a, bf(h), bf(h), bf(r), bf(nw), T, 1e-6f);
    qwen::linear_w4a8(bf(mid), wu, a, T, nullptr, QW4_ACT_SWIGLU, nullptr, ws);
    qwen::quantize_a8(b, bf(mid), I, T);
    qwen::a8_dequant_rows(bf(back), b, 0, T);
    qwen::linear_w4a8(bf(out), wd, b, T, nullptr, QW4_ACT_NONE, bf(h), ws);
    qwen::linear_w4a8_f32(logits.p, wh, a, T, ws);
    qwen::logprobs_f32(lp.p, ent.p, ids.p, top.p, logits.p, V, targets.p, T, V, asked, k, ws);
    CK(hipDeviceSynchronize());
    const std::vector<double> xa = held(a, T), xb = held(b, T), m = doubles(mid), o = doubles(out), sum = doubles(h);
    std::vector<double> want((size_t)T * H);
    for (int t = 0; t < T; ++t) {
      double ss = 0;
      for (int i = 0; i < H; ++i) {
        const size_t at = (size_t)t * H + i;
        if (or_f32_to_bf16(or_bf16_to_f32(h0[at]) + or_bf16_to_f32(r0[at])) != or_f32_to_bf16((float)sum[at])) ++cn.bad;
        ss += sum[at] * sum[at];
      }
      for (int i = 0; i < H; ++i)
        want[(size_t)t * H + i] = sum[(size_t)t * H + i] / std::sqrt(ss / H + 1e-6) * (1 + (double)or_bf16_to_f32(norm_w[i]));
    }
    codes(cn, want, xa, 32 * 0x1p-24);   // the norm's fp32: some 24 roundings of the sum, halved, and 10
    codes(cq, m, xb, 0);
    const std::vector<double> bk = doubles(back);
    for (size_t i = 0; i < bk.size(); ++i) cb(bk[i], xb[i], (0x1p-8 + 0x1p-24) * std::fabs(xb[i]));
    for (int t = 0; t < T; ++t) {
      double s1, s2;
      for (int i = 0; i < I; ++i) {
        const double g = dot(up, xa, i, t, H, s1), u = dot(up, xa, I + i, t, H, s2), f = g / (1 + std::exp(-g));
        const double tg = sum_bound(s1, H), tu = sum_bound(s2, H);
        // silu's slope is below 1.1; exp's argument |g| 2^-24, its and the quotient's steps 20
        const double off = 1.1 * tg * (std::fabs(u) + tu) + std::fabs(f) * tu + (std::fabs(g) + 20) * 0x1p-23 * std::fabs(f * u);
        cu(m[(size_t)t * I + i], f * u, off + (0x1p-8 + 0x1p-23) * std::fabs(f * u) + 0x1p-8 * off);
      }
      for (int n = 0; n < H; ++n) {
        const double v = dot(down, xb, n, t, I, s1) + sum[(size_t)t * H + n];
        const double off = sum_bound(s1, I) + 0x1p-24 * std::fabs(v);
        cd(o[(size_t)t * H + n], v, off + (0x1p-8 + 0x1p-23) * std::fabs(v) + 0x1p-8 * off);
      }
    }
    const std::vector<float> lg = logits.host(), glp = lp.host(), gent = ent.host(), gtop = top.host();
    const std::vector<int32_t> gid = ids.host();
    for (int t = 0; t < T; ++t) {
      double size;
      for (int n = 0; n < V; ++n) {
        const double v = dot(head, xa, n, t, H, size);
        cl(lg[(size_t)t * V + n], v, sum_bound(size, H));
      }
      const float* x = &lg[(size_t)t * V];
      const double hi = *std::max_element(x, x + V), lo = *std::min_element(x, x + V);
      double L = 0, e = 0;
      for (int n = 0; n < V; ++n) L += std::exp(x[n] - hi);
      L = hi + std::log(L);
      for (int n = 0; n < V; ++n) e -= std::exp(x[n] - L) * (x[n] - L);
      // x - m, and that less the log: half a step of the range each; the log's own few steps
      const double step = 0x1p-24 * (2 * (hi - lo) + 64);
      ce(gent[t], e, 64 * 0x1p-24 * (1 + std::log((double)V)));
      for (int j = 0; j < asked; ++j) {
        const int id = ask[(size_t)t * asked + j];
        cp(glp[(size_t)t * asked + j], id < V ? x[id] - L : 0, id < V ? step : 0);
      }
      std::vector<int> order(V);
      for (int n = 0; n < V; ++n) order[n] = n;
      std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return x[i] > x[j]; });
      for (int j = 0; j < k; ++j) {
        ci(gid[(size_t)t * k + j], order[j], 0);
        ct(gtop[(size_t)t * k + j], x[order[j]] - L, step);
      }
    }
  }
  bool ok = true;
  for (const Check* c : {&cn, &cu, &cq, &cd, &cb, &cl, &cp, &ce, &ct, &ci}) ok = c->ok() && ok;
  qwen::a8_free(a);
  qwen::a8_free(b);
  qwen::gemm_workspace_free(ws);
  for (qwen::W4A16Weights* w : {&wu, &wd, &wh}) qwen::awq_free(*w);
  std::printf(ok ? "gate_a8_values: PASS\n" : "gate_a8_values: FAIL\n");
  return ok ? 0 : 1;
}
