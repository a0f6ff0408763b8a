// The steps either side of the products grouped by expert: the router (top-k of a
// token's logits, softmax weights, and the plan that groups the (token, slot)
// pairs by expert) and the weighted sum of a token's expert rows. No reference
// counterpart: its model is dense.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../../include/qwen_w4a16.h"
#include "grouped.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

static_assert(kMaxExperts == 1024, "16 logits a lane");
constexpr int kMaxTopK = 16;        // a row of 16 lanes holds a token's choice
// Pairs that one workgroup plans: a thread each, whose place among its expert's pairs is
// counted over all pairs before it (256 pairs: 1.5 us slower than k_plan).
constexpr int kSmallPairs = 128;
// Tokens of such a plan that it routes as well, in a single launch, a wave each (32 tokens
// over 128 experts: 11.7 us, in two launches 7.0; 16 over 64: 6.8 and 6.9).
constexpr int kSmallTokens = 16;

struct PlanArgs {
  int32_t *offsets, *tokens, *pos;   // offsets null: no plan wanted
};

struct RouteArgs {
  const void* logits;
  int32_t* ids;
  float* weights;
  PlanArgs plan;
  int T, E, k, renorm;
};

// Order-preserving key of a logit: larger key, larger value. -0 counts as +0, and
// NaN and -Inf, which no token chooses, are 0.
__device__ __forceinline__ uint32_t logit_key(float v) {
  v = v == 0.f ? 0.f : v;
  const uint32_t u = __float_as_uint(v);
  return v > -__builtin_inff() ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// Reductions over a wave: the 16 lanes of a DPP row (xor 1, xor 2, half-row mirror,
// row mirror), then the four rows through scalar registers.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, dpp<0xB1>(v));
  v = max(v, dpp<0x4E>(v));
  v = max(v, dpp<0x141>(v));
  v = max(v, dpp<0x140>(v));
  const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}
__device__ __forceinline__ float row16_add(float v) {
  v += __uint_as_float(dpp<0xB1>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x4E>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x140>(__float_as_uint(v)));
  return v;
}
__device__ __forceinline__ float lane_value(float v, int l) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l));
}
__device__ __forceinline__ float wave_add(float v) {
  v = row16_add(v);
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}

__device__ __forceinline__ int wave_add_int(int v) {
  v += (int)dpp<0xB1>((uint32_t)v);
  v += (int)dpp<0x4E>((uint32_t)v);
  v += (int)dpp<0x141>((uint32_t)v);
  v += (int)dpp<0x140>((uint32_t)v);
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

template <class T>
__device__ __forceinline__ float logit(const T* p) {
  if constexpr (std::is_same_v<T, float>)
    return *p;
  else
    return bf16_bits_to_f32(*p);
}

// One wave chooses the experts of row t. Lane l holds the logits l PER .. l PER +
// PER - 1 as keys; each of the k rounds takes the wave's largest key, from the lowest
// lane that holds it (so ties go to the lowest expert), and strikes it out there.
// Lane j < 16 returns slot j: expert (-1: none left) and weight.
template <class T, int PER>
__device__ __forceinline__ void route_row(const RouteArgs& a, int t, int lane, int& id, float& weight) {
  const T* row = static_cast<const T*>(a.logits) + (size_t)t * a.E;
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    key[i] = e < a.E ? logit_key(logit(row + e)) : 0u;
  }
  uint32_t best = 0;
  int at = 0;
  auto look = [&] {
    best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
  };
  look();
  // exp(v - largest); +Inf logits share the whole weight
  const uint32_t top = wave_max(best);
  const float vtop = key_value(top);
  auto mass = [&](uint32_t k) {
    const float v = key_value(k);
    if (k == 0u) return 0.f;
    return v == vtop ? 1.f : expf(v - vtop);
  };
  float total = 0.f;
  if (!a.renorm) {
#pragma unroll
    for (int i = 0; i < PER; ++i) total += mass(key[i]);
    total = wave_add(total);
  }
  id = -1;
  uint32_t mine = 0;
  for (int j = 0; j < a.k; ++j) {
    const uint32_t m = j == 0 ? top : wave_max(best);
    if (m == 0u) break;
    const int from = __builtin_ctzll(__ballot(best == m));
    const int e = from * PER + __builtin_amdgcn_readlane(at, from);
    if (lane == j) {
      id = e;
      mine = m;
    }
    if (lane == from) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i == at) key[i] = 0u;
      look();
    }
  }
  const float p = mass(mine);
  if (a.renorm) total = row16_add(lane < kMaxTopK ? p : 0.f);
  weight = id >= 0 ? p / total : 0.f;
}

template <class T, int PER>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= a.T) return;
  int id;
  float w;
  route_row<T, PER>(a, t, lane, id, w);
  if (lane < a.k) {
    a.ids[(size_t)t * a.k + lane] = id;
    a.weights[(size_t)t * a.k + lane] = w;
  }
}

// The plan of R <= kSmallPairs pairs by one workgroup of 64 W threads, at least E and
// R, from their experts in LDS: a histogram (integer atomics: any order gives the same counts), its
// running sum, and for each pair the earlier pairs of its expert counted.
template <int W>
struct SmallPlan {
  int ids[kSmallPairs];
  int start[64 * W];
  int wsum[W];
};
template <int W>
__device__ __forceinline__ void plan_small(const PlanArgs& p, SmallPlan<W>& s, int R, int E, int k) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  s.start[t] = 0;   // one entry per thread
  __syncthreads();
  const int id = t < R ? s.ids[t] : -1;
  const bool live = (unsigned)id < (unsigned)E;
  if (live) atomicAdd(&s.start[id], 1);
  __syncthreads();
  const int n = s.start[t];
  int sum = n;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(sum, off, 64);
    if (lane >= off) sum += v;
  }
  if (lane == 63) s.wsum[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int v = s.wsum[w];
    before += w < wave ? v : 0;
    all += v;
  }
  const int first = before + sum - n;
  s.start[t] = first;
  if (t < E) p.offsets[t] = first;
  if (t == 0) p.offsets[E] = all;
  __syncthreads();
  if (t < R) {
    int rank = 0;
    for (int i = 0; i < t; ++i) rank += s.ids[i] == id;
    const int at = live ? s.start[id] + rank : -1;
    p.pos[t] = at;
    if (live) p.tokens[at] = t / k;
    if (t >= all) p.tokens[t] = -1;
  }
}

// Few tokens: choice and plan in one launch. A decoded token's router is all latency,
// and a second launch would add as much again; of few waves where they do (4 instead of
// 16, one token over 64 experts: 3.8 us instead of 4.0).
template <class T, int PER, int W>
__global__ __launch_bounds__(64 * W) void k_route_small(RouteArgs a) {
  __shared__ SmallPlan<W> s;
  const int lane = threadIdx.x & 63;
  for (int t = threadIdx.x >> 6; t < a.T; t += W) {
    int id;
    float w;
    route_row<T, PER>(a, t, lane, id, w);
    if (lane < a.k) {
      a.ids[t * a.k + lane] = id;
      a.weights[t * a.k + lane] = w;
      s.ids[t * a.k + lane] = id;
    }
  }
  __syncthreads();
  plan_small(a.plan, s, a.T * a.k, a.E, a.k);
}

__global__ __launch_bounds__(1024) void k_plan_small(PlanArgs p, const int32_t* ids, int R, int E, int k) {
  __shared__ SmallPlan<16> s;
  if ((int)threadIdx.x < R) s.ids[threadIdx.x] = ids[threadIdx.x];
  __syncthreads();
  plan_small(p, s, R, E, k);
}

// The plan of many pairs: workgroup e gathers expert e's pairs, in order. Wave w takes
// the w-th sixteenth of the pairs' experts, kPlanAhead loads of 256 at once, four pairs a
// lane: first it counts those below e (they come before e's first position) and those equal
// to e, then it gives the equal ones their places; up to 16 x 256 kPlanAhead pairs stay in
// registers in between. No workgroup waits for another. Bound by the instructions of a
// workgroup's 16 waves: 32768 pairs of 128 experts 22.2 us with a load at a time, 11.5 with
// all in flight, 9.4 without a division for every hit, 8.0 with four pairs a load.
constexpr int kPlanAhead = 8;

__global__ __launch_bounds__(1024) void k_plan(PlanArgs p, const int32_t* ids, int R, int E, int k) {
  __shared__ int below[16], equal[16];
  const int e = blockIdx.x, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seg = ((R - 1) / 4096 + 1) * 256;   // pairs of a wave, in whole loads
  const long long first = (long long)wave * seg;
  const int i0 = (int)std::min<long long>(first, R), i1 = (int)std::min<long long>(first + seg, R);
  typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int kRound = 256 * kPlanAhead;
  int id[kPlanAhead][4];   // pair i + 256 r + 4 lane + c
  auto load = [&](int i) __attribute__((always_inline)) {
    auto four = [&](int r) __attribute__((always_inline)) {
      const i32x4 v = *reinterpret_cast<const i32x4*>(ids + i + 256 * r + 4 * lane);
#pragma unroll
      for (int c = 0; c < 4; ++c) id[r][c] = v[c];
    };
    if (i1 - i >= kRound) {   // without a branch a load
#pragma unroll
      for (int r = 0; r < kPlanAhead; ++r) four(r);
      return;
    }
#pragma unroll
    for (int r = 0; r < kPlanAhead; ++r) {
      const int left = i1 - i - 256 * r;   // wave-uniform
      if (left >= 256) {
        four(r);
        continue;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        id[r][c] = -1;
        if (left > 0 && 4 * lane + c < left) id[r][c] = ids[i + 256 * r + 4 * lane + c];
      }
    }
  };
  const bool kept = i1 - i0 <= kRound;
  int nb = 0, ne = 0;
  for (int i = i0; i < i1; i += kRound) {
    load(i);
#pragma unroll
    for (int r = 0; r < kPlanAhead; ++r) {
      if (i1 - i <= 256 * r) break;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        nb += (unsigned)id[r][c] < (unsigned)e;
        ne += (int)__popcll(__ballot(id[r][c] == e));
      }
    }
    if (i1 - i <= kRound) break;   // no overflow of i
  }
  nb = wave_add_int(nb);
  if (lane == 0) {
    below[wave] = nb;
    equal[wave] = ne;
  }
  __syncthreads();
  int start = 0, at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    start += below[w];
    at += w < wave ? equal[w] : 0;
    total += equal[w];
  }
  at += start;
  if (threadIdx.x == 0) {
    p.offsets[e] = start;
    if (e == E - 1) p.offsets[E] = start + total;
  }
  // x / k = x inv / 2^16 for x < kRound + k: inv k - 2^16 < k <= 16 moves it by x / 2^16 < 1 / k
  const uint32_t inv = (65536u + (uint32_t)k - 1u) / (uint32_t)k;
  static_assert((kRound + kMaxTopK) * kMaxTopK < 65536, "exact");
  for (int i = i0; i < i1; i += kRound) {
    if (!kept) load(i);
    const int tok0 = i / k;
    const uint32_t x0 = (uint32_t)(i - tok0 * k + 4 * lane);
#pragma unroll
    for (int r = 0; r < kPlanAhead; ++r) {
      if (i1 - i <= 256 * r) break;
      unsigned long long hit[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) hit[c] = __ballot(id[r][c] == e);
      if (hit[0] | hit[1] | hit[2] | hit[3]) {   // wave-uniform
        int to = at;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          to = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(hit[c] >> 32),
                                              __builtin_amdgcn_mbcnt_lo((uint32_t)hit[c], (uint32_t)to));
          at += (int)__popcll(hit[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (id[r][c] == e) {
            p.tokens[to] = tok0 + (int)((x0 + 256u * r + c) * inv >> 16);
            p.pos[i + 256 * r + 4 * lane + c] = to;
            ++to;
          }
      }
    }
    if (e == 0) {   // the pairs of no expert
#pragma unroll
      for (int r = 0; r < kPlanAhead; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int left = i1 - i - 256 * r;
          if (4 * lane + c < left && (unsigned)id[r][c] >= (unsigned)E) p.pos[i + 256 * r + 4 * lane + c] = -1;
        }
    }
    if (i1 - i <= kRound) break;
  }
  if (e == E - 1)
    for (int i = start + total + threadIdx.x; i < R; i += 1024) p.tokens[i] = -1;
}

// out[t] = bf16(residual[t] + sum_j weights[t][j] y[pos[t][j]]), the terms added in
// fp32 in slot order. A thread sums 8 columns; a token's positions and weights are the
// same for its whole workgroup (scalar loads), and the rows' loads go out together.
constexpr int kCombineThreads = 256;
constexpr int kCombineAhead = 8;

__global__ __launch_bounds__(kCombineThreads) void k_combine(uint16_t* out, const uint16_t* y,
                                                             const int32_t* pos, const float* weights,
                                                             const uint16_t* residual, int R, int k,
                                                             int chunks) {
  const int t = blockIdx.x;
  const int i = blockIdx.y * kCombineThreads + threadIdx.x;
  if (i >= chunks) return;
  const size_t at = (size_t)t * chunks + i;
  float acc[8];
  u32x4 r = {0u, 0u, 0u, 0u};
  if (residual) r = reinterpret_cast<const u32x4*>(residual)[at];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    acc[2 * c] = bf16_bits_to_f32(r[c] & 0xffffu);
    acc[2 * c + 1] = bf16_bits_to_f32(r[c] >> 16);
  }
  const u32x4* rows = reinterpret_cast<const u32x4*>(y);
  for (int j0 = 0; j0 < k; j0 += kCombineAhead) {
    u32x4 v[kCombineAhead];
    float w[kCombineAhead];
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j) {
      int p = -1;
      w[j] = 0.f;
      if (j0 + j < k) {
        p = pos[(size_t)t * k + j0 + j];
        w[j] = weights[(size_t)t * k + j0 + j];
      }
      v[j] = u32x4{0u, 0u, 0u, 0u};
      if ((unsigned)p < (unsigned)R)
        v[j] = rows[(size_t)p * chunks + i];
      else
        w[j] = 0.f;   // no row: nothing, whatever its weight
    }
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[2 * c] = __builtin_fmaf(w[j], bf16_bits_to_f32(v[j][c] & 0xffffu), acc[2 * c]);
        acc[2 * c + 1] = __builtin_fmaf(w[j], bf16_bits_to_f32(v[j][c] >> 16), acc[2 * c + 1]);
      }
  }
  u32x4 o;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] = pack_bf16x2(acc[2 * c], acc[2 * c + 1]);
  reinterpret_cast<u32x4*>(out)[at] = o;
}

int check_plan(const qw4_plan* p, long long pairs) {
  if (!p || !p->offsets || (pairs > 0 && (!p->tokens || !p->pos))) return QW4_ERR_NULL;
  if (p->experts < 1 || p->experts > kMaxExperts) return QW4_ERR_SHAPE;
  if (pairs > p->max_pairs) return QW4_ERR_SCRATCH;
  return QW4_OK;
}

void launch_plan(const PlanArgs& p, const int32_t* ids, int R, int E, int k, hipStream_t s) {
  if (R <= kSmallPairs)
    k_plan_small<<<1, 1024, 0, s>>>(p, ids, R, E, k);
  else
    k_plan<<<E, 1024, 0, s>>>(p, ids, R, E, k);
}

template <class T, int PER>
void launch_route(const RouteArgs& a, hipStream_t s) {
  if (a.plan.offsets && a.T <= kSmallTokens && a.T * a.k <= kSmallPairs) {
    if (PER <= 4 && a.T <= 4)
      k_route_small<T, PER, 4><<<1, 256, 0, s>>>(a);
    else
      k_route_small<T, PER, 16><<<1, 1024, 0, s>>>(a);
    return;
  }
  launch_rows_of(a.T, 1 << 24, [&](int first, int n) {
    RouteArgs r = a;
    r.logits = static_cast<const T*>(a.logits) + (size_t)first * a.E;
    r.ids += (size_t)first * a.k;
    r.weights += (size_t)first * a.k;
    r.T = n;
    if (n > 0) k_route<T, PER><<<(n + 3) / 4, 256, 0, s>>>(r);
  });
  if (a.plan.offsets) launch_plan(a.plan, a.ids, a.T * a.k, a.E, a.k, s);
}

template <class T>
int route(int32_t* ids, float* weights, const qw4_plan* plan, const T* logits, int T_, int E, int k,
          int renorm, void* stream) {
  if (T_ < 0) return QW4_ERR_M;
  if (E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E) return QW4_ERR_SHAPE;
  const long long pairs = (long long)T_ * k;
  if (pairs > 0x7fffffffLL - 2048) return QW4_ERR_SHAPE;
  if (T_ > 0 && (!ids || !weights || !logits)) return QW4_ERR_NULL;
  RouteArgs a{logits, ids, weights, {}, T_, E, k, renorm};
  if (plan) {
    const int st = check_plan(plan, pairs);
    if (st) return st;
    if (plan->experts != E) return QW4_ERR_SHAPE;
    a.plan = {plan->offsets, plan->tokens, plan->pos};
  }
  if (T_ == 0 && !plan) return QW4_OK;
  hipStream_t s = (hipStream_t)stream;
  if (E <= 64)
    launch_route<T, 1>(a, s);
  else if (E <= 128)
    launch_route<T, 2>(a, s);
  else if (E <= 256)
    launch_route<T, 4>(a, s);
  else if (E <= 512)
    launch_route<T, 8>(a, s);
  else
    launch_route<T, 16>(a, s);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_plan_alloc(qw4_plan* p, int experts, int max_pairs) {
  if (!p) return QW4_ERR_NULL;
  std::memset(p, 0, sizeof(*p));
  if (experts < 1 || experts > kMaxExperts || max_pairs < 1) return QW4_ERR_SHAPE;
  qw4_plan q{};
  hipError_t e = hipMalloc(&q.offsets, ((size_t)experts + 1) * 4);
  if (e == hipSuccess) e = hipMalloc(&q.tokens, (size_t)max_pairs * 4);
  if (e == hipSuccess) e = hipMalloc(&q.pos, (size_t)max_pairs * 4);
  if (e != hipSuccess) {
    set_hip_error((int)e);
    (void)hipGetLastError();
    if (q.offsets) (void)hipFree(q.offsets);
    if (q.tokens) (void)hipFree(q.tokens);
    return QW4_ERR_NOMEM;
  }
  q.experts = experts;
  q.max_pairs = max_pairs;
  *p = q;
  return QW4_OK;
}

int qw4_plan_free(qw4_plan* p) {
  if (!p) return QW4_ERR_NULL;
  if (p->offsets) (void)hipFree(p->offsets);
  if (p->tokens) (void)hipFree(p->tokens);
  if (p->pos) (void)hipFree(p->pos);
  std::memset(p, 0, sizeof(*p));
  return QW4_OK;
}

int qw4_route(int32_t* ids, float* weights, const qw4_plan* plan, const uint16_t* logits, int T,
              int experts, int top_k, int renorm, void* stream) {
  return route<uint16_t>(ids, weights, plan, logits, T, experts, top_k, renorm, stream);
}

int qw4_route_f32(int32_t* ids, float* weights, const qw4_plan* plan, const float* logits, int T,
                  int experts, int top_k, int renorm, void* stream) {
  return route<float>(ids, weights, plan, logits, T, experts, top_k, renorm, stream);
}

int qw4_route_ids(const qw4_plan* plan, const int32_t* ids, int T, int top_k, void* stream) {
  if (T < 0) return QW4_ERR_M;
  if (top_k < 1 || top_k > kMaxTopK) return QW4_ERR_SHAPE;
  const long long pairs = (long long)T * top_k;
  if (pairs > 0x7fffffffLL - 2048) return QW4_ERR_SHAPE;
  if (T > 0 && !ids) return QW4_ERR_NULL;
  const int st = check_plan(plan, pairs);
  if (st) return st;
  launch_plan({plan->offsets, plan->tokens, plan->pos}, ids, (int)pairs, plan->experts, top_k,
              (hipStream_t)stream);
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

int qw4_combine(uint16_t* out, const uint16_t* y, const qw4_plan* plan, const float* weights, int T,
                int top_k, int dim, const uint16_t* residual, void* stream) {
  if (T < 0) return QW4_ERR_M;
  if (top_k < 1 || top_k > kMaxTopK || dim <= 0 || dim % 8) return QW4_ERR_SHAPE;
  const long long pairs = (long long)T * top_k;
  const long long cols = (dim / 8 + kCombineThreads - 1) / kCombineThreads;
  if (pairs > 0x7fffffffLL - 2048 || cols > 65535) return QW4_ERR_SHAPE;
  const int st = check_plan(plan, pairs);
  if (st) return st;
  if (T == 0) return QW4_OK;
  if (!out || !y || !weights) return QW4_ERR_NULL;
  if (((uintptr_t)out | (uintptr_t)y | (uintptr_t)residual) & 15) return QW4_ERR_ALIGN;
  launch_rows_of(T, 1 << 23, [&](int first, int n) {
    const size_t at = (size_t)first * dim, pair = (size_t)first * top_k;
    k_combine<<<dim3(n, (unsigned)cols), kCombineThreads, 0, (hipStream_t)stream>>>(
        out + at, y, plan->pos + pair, weights + pair, residual ? residual + at : nullptr, (int)pairs, top_k,
        dim / 8);
  });
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // extern "C"
