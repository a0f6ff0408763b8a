// Log probabilities of given tokens, entropy and top alternatives of rows of logits, in
// one pass over each row.
//
// A wave streams blocks of 512 logits, 8 a lane, and keeps
//   m       the largest so far (the same in all lanes),
//   s       per lane, sum of exp(x - m) without the one element that is m (`own`: it was
//           this lane's),
//   u       per lane, sum of exp(x - m) (x - m).
// With total = 1 + s:  L = m + log1p(s),  H = log1p(s) - u / (1 + s). Without the
// largest element s keeps its relative precision when that token is all but certain,
// where 1 + s would lose it and both results are about s.
// All of it in fp32: a lane sums n / (256 S) terms, S the splits of the row, the joins some 16,
// so that s is off by (n / 256 + 80) 2^-24 of itself at most, by some 1e-7 in fact; sums in 64 bits
// come 1.5 to 4 times as near, which logits of 8 or 24 bits have no use for.
//
// Alternatives: a lane keeps the six largest maxima of its eights as keys (the upper 16
// bits of the value, ordered, over the block's number): 2 vector instructions a logit,
// no branch. At the end the k-th largest of the lanes' first keys bounds the k-th largest
// logit from below, and one wave reads the eights whose key reaches it again, some k of them.
// Where a lane's sixth key reaches it, there may have been a seventh: then the waves go over
// their blocks once more and keep lists (sorted or constant rows). 1000 x 248320 bf16 logits
// take 102 us at k = 5, 20 and 32, and 92 without alternatives; with lists kept from the start
// they took 138 / 207 / 245; with four keys one row of some 500 went over its blocks again at
// k = 32, and its workgroup alone lengthened the launch to 212 us (five: 149).
//
// Rows split over workgroups, for few rows, write (m, s, u, list) to the workspace and
// a second kernel joins them in order; nothing depends on which workgroup comes first.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/qwen_w4a16.h"
#include "w4a16_common.h"

namespace qw4 {
namespace {

constexpr int kLpMaxTop = 32;
constexpr int kLpWaves = 4;
constexpr int kLpBlock = 512;    // logits of a wave's block
constexpr int kLpAhead = 4;      // blocks in flight
constexpr int kLpFew = 12;       // entries put into a list one by one

struct LpArgs {
  const void* x;
  size_t ld;
  const int32_t* targets;
  float *lp, *entropy, *top_lp;
  int32_t* top_ids;
  int n, asked, k, S;
  int few;             // a wave's blocks are fewer than 2^16, the row's than 2^24
  uint32_t* part;      // [T][S] records of 4 + 2 k words
};

struct LpStats {
  float m, s, u;       // s, u: of the whole wave once joined
};

__device__ __forceinline__ float lane_value(float v, int l) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// v of lane (lane ^ X), in registers (through LDS, as shuffles go, a step of the networks
// below waits 5 times as long).
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  if constexpr (X == 1) return dpp<0xB1>(v);                // quad_perm [1, 0, 3, 2]
  if constexpr (X == 2) return dpp<0x4E>(v);                // quad_perm [2, 3, 0, 1]
  if constexpr (X == 4) return dpp<0x1B>(dpp<0x141>(v));    // half rows mirrored, fours mirrored
  if constexpr (X == 8) return dpp<0x128>(v);               // rows rotated by 8
  if constexpr (X == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? p[0] : p[1];
  }
  if constexpr (X == 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? p[0] : p[1];
  }
}
template <int X>
__device__ __forceinline__ float lane_xor(float v, int lane) {
  return __uint_as_float(lane_xor<X>(__float_as_uint(v), lane));
}
__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += lane_xor<1>(v, lane);
  v += lane_xor<2>(v, lane);
  v += lane_xor<4>(v, lane);
  v += lane_xor<8>(v, lane);
  v += lane_xor<16>(v, lane);
  return v + lane_xor<32>(v, lane);
}
__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, lane_xor<1>(v, lane));
  v = fmaxf(v, lane_xor<2>(v, lane));
  v = fmaxf(v, lane_xor<4>(v, lane));
  v = fmaxf(v, lane_xor<8>(v, lane));
  v = fmaxf(v, lane_xor<16>(v, lane));
  return lane_value(fmaxf(v, lane_xor<32>(v, lane)), 0);
}
// exp(d), d <= 0; its argument's rounding, |d| 2^-24, is the d's own.
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.4426950408889634f); }
// A difference to multiply with: e^-10000 is 0, and 0 times it stays 0.
__device__ __forceinline__ float lp_far(float d) { return fmaxf(d, -10000.f); }

// The sums of reference m (own of them the element m itself, 0 or 1) under reference to >= m.
__device__ __forceinline__ void lp_rescale(float& s, float& u, float own, float m, float to) {
  const float d = lp_far(m - to), c = lp_exp(d), all = s + own;
  u = c * (u + d * all);
  s = c * all;
}

// A larger value, then a lower index, comes first; -Inf (no token) last.
__device__ __forceinline__ bool lp_first(float v, int i, float w, int j) {
  return v > w || (v == w && (unsigned)i < (unsigned)j);
}

// The best of what a wave has seen, lane j the j-th of 64.
struct LpList {
  float v = -INFINITY;
  int i = -1;

  // One step of a bitonic network: a lane and its partner STRIDE off keep the first
  // (upper) or the other of their two entries.
  template <int STRIDE>
  __device__ __forceinline__ void exchange(bool upper, int lane) {
    const float w = lane_xor<STRIDE>(v, lane);
    const int j = (int)lane_xor<STRIDE>((uint32_t)i, lane);
    if (lp_first(v, i, w, j) != upper) {
      v = w;
      i = j;
    }
  }
  // Steps of strides STRIDE, STRIDE / 2, ... 1 within runs of SIZE entries, every other run
  // the other way round.
  template <int SIZE, int STRIDE>
  __device__ __forceinline__ void runs(int lane) {
    exchange<STRIDE>((SIZE == 64 || (lane & SIZE) == 0) == ((lane & STRIDE) == 0), lane);
    if constexpr (STRIDE > 1) runs<SIZE, STRIDE / 2>(lane);
  }
  __device__ __forceinline__ void settle(int lane) { runs<64, 32>(lane); }   // sorts a bitonic sequence
  __device__ __forceinline__ void sort(int lane) {
    runs<2, 1>(lane);
    runs<4, 2>(lane);
    runs<8, 4>(lane);
    runs<16, 8>(lane);
    runs<32, 16>(lane);
    settle(lane);
  }
  // The best 64 of this sorted list and another.
  __device__ __forceinline__ void merge(const LpList& o, int lane) {
    const float w = __shfl(o.v, 63 - lane, 64);   // reversed
    const int j = __shfl(o.i, 63 - lane, 64);
    if (lp_first(w, j, v, i)) {
      v = w;
      i = j;
    }
    settle(lane);
  }
  // One entry (the same in all lanes) into its place.
  __device__ __forceinline__ void insert(float x, int at, int lane) {
    const int c = __popcll(__ballot(lp_first(v, i, x, at)));
    // wave_shr:1, the lane below's
    const float pv = __uint_as_float(
        (uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x138, 0xf, 0xf, false));
    const int pi = __builtin_amdgcn_update_dpp(0, i, 0x138, 0xf, 0xf, false);
    if (lane >= c) {
      v = lane == c ? x : pv;
      i = lane == c ? at : pi;
    }
  }
};

struct LpSlot {
  float v;
  int i;
};

constexpr int kLpKeys = 6;   // eights that a lane remembers

// A maximum's order in 16 bits (larger: larger, or equal up to the bits cut off; -Inf and
// below: at most kLpNone), and the least value of that order.
constexpr uint32_t kLpNone = 0x7f;
__device__ __forceinline__ uint32_t lp_order(float v) {
  const int b = __float_as_int(v + 0.f);   // -0 as 0
  return (uint32_t)(b ^ ((b >> 31) | (int)0x80000000)) >> 16;
}
__device__ __forceinline__ float lp_least(uint32_t order) {
  const uint32_t u = order << 16;
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <bool TOP>
struct LpWave {
  float m = -INFINITY;
  float s = 0.f, u = 0.f, own = 0.f;
  uint32_t key[kLpKeys] = {};   // descending
  LpList list;
  float last = -INFINITY;       // the list's k-th entry, which another has to beat
  int last_i = -1;

  // Elements x[e] of the lane (-Inf where there is none): their share of the sums, and their
  // maximum.
  template <int N>
  __device__ __forceinline__ float add(const float (&x)[N], int lane) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, x[e]);
    if (__ballot(top > m)) {
      const float to = wave_max(top, lane);
      lp_rescale(s, u, own, m, to);
      m = to;
      bool mine = lane == __builtin_ctzll(__ballot(top == to));
      own = mine ? 1.f : 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = x[e] - m, p = lp_exp(d);
        if (mine && x[e] == to) {
          mine = false;   // m itself stays out of s
        } else {
          s += p;
          u = __builtin_fmaf(p, lp_far(d), u);
        }
      }
      return top;
    }
    const float ref = m > -INFINITY ? m : 0.f;   // nothing but -Inf so far: they add nothing
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - ref, p = lp_exp(d);
      s += p;
      u = __builtin_fmaf(p, lp_far(d), u);
    }
    return top;
  }

  __device__ __forceinline__ void remember(float top, uint32_t number) {
    const uint32_t k = (lp_order(top) << 16) | number;
#pragma unroll
    for (int l = kLpKeys - 1; l > 0; --l) key[l] = max(key[l], min(key[l - 1], k));
    key[0] = max(key[0], k);
  }

  __device__ __forceinline__ void close(int k) {
    last = lane_value(list.v, k - 1);
    last_i = __builtin_amdgcn_readlane(list.i, k - 1);
  }

  // Elements x[e] with indices at(e), rising with e, into the list: while that is empty,
  // only those from `least` on, which k are at least. Many at once are gathered and sorted, a
  // few put in one by one.
  template <int N, class At>
  __device__ __forceinline__ void choose(const float (&x)[N], const At& at, int k, int lane, float least,
                                         LpSlot* slots) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, x[e]);
    if (!__ballot(top >= last && top > -INFINITY)) return;
    auto wanted = [&](float v, int i) { return v >= least && v > -INFINITY && lp_first(v, i, last, last_i); };
    int count = 0, mine[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const unsigned long long some = __ballot(wanted(x[e], at(e)));
      mine[e] = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
      count += __popcll(some);
    }
    if (count > kLpFew && count <= 64) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (wanted(x[e], at(e))) slots[mine[e]] = {x[e], at(e)};
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      LpList more;
      if (lane < count) {
        more.v = slots[lane].v;
        more.i = slots[lane].i;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      more.sort(lane);
      if (last > -INFINITY || lane_value(list.v, 0) > -INFINITY)
        list.merge(more, lane);
      else
        list = more;
      close(k);
      return;
    }
    uint32_t done = 0;   // elements of this lane that are in the list
    for (;;) {
      float b = -INFINITY;
      int bi = -1, be = 0;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!(done >> e & 1) && x[e] > b) {
          b = x[e];
          bi = at(e);
          be = e;
        }
      const unsigned long long some = __ballot(wanted(b, bi));
      if (!some) break;
      const int from = __builtin_ctzll(some);
      list.insert(lane_value(b, from), __builtin_amdgcn_readlane(bi, from), lane);
      close(k);
      if (lane == from) done |= 1u << be;
    }
  }

  // The k-th largest of the lanes' `top` while the list is empty.
  __device__ __forceinline__ float first_least(float top, int k, int lane) const {
    if (lane_value(list.v, 0) > -INFINITY) return -INFINITY;
    int rank = 0;
    for (int l = 0; l < 64; ++l) {
      const float o = lane_value(top, l);
      rank += o > top || (o == top && l < lane);
    }
    return wave_max(rank == k - 1 ? top : -INFINITY, lane);
  }

  __device__ __forceinline__ LpStats stats(int lane) const { return {m, wave_sum(s, lane), wave_sum(u, lane)}; }
};

// The statistics of two disjoint sets: the largest of both stays out of s once.
__device__ __forceinline__ LpStats lp_join(LpStats a, LpStats b) {
  if (b.m > a.m) {
    const LpStats t = a;
    a = b;
    b = t;
  }
  lp_rescale(b.s, b.u, b.m > -INFINITY ? 1.f : 0.f, b.m, a.m);
  return {a.m, a.s + b.s, a.u + b.u};
}

template <class T>
__device__ __forceinline__ float lp_logit(const T* p) {
  if constexpr (std::is_same_v<T, float>)
    return *p;
  else
    return bf16_bits_to_f32(*p);
}

// Target j of a row and its logit, where there is one.
struct LpAsked {
  bool in;
  float x;
};
template <class T>
__device__ __forceinline__ LpAsked lp_asked(const LpArgs& a, int row, int j) {
  if (j >= a.asked) return {false, 0.f};
  const int i = a.targets[(size_t)row * a.asked + j];
  const bool in = (unsigned)i < (unsigned)a.n;
  return {in, in ? lp_logit(static_cast<const T*>(a.x) + (size_t)row * a.ld + i) : 0.f};
}

// A row's results from its statistics and list, by one wave; `first` is target `lane`.
template <class T>
__device__ __forceinline__ void lp_write(const LpArgs& a, int row, LpStats t, const LpList& list, LpAsked first,
                                         int lane) {
  const bool some = t.m > -INFINITY;
  if (t.m == INFINITY) t.s = __builtin_nanf("");
  const float log = some ? log1pf(t.s) : t.s;   // of a row without any: 0, or NaN
  if (lane == 0 && a.entropy) a.entropy[row] = some ? log - t.u / (1.f + t.s) : log;
  auto lp = [&](float x) { return (some ? x - t.m : -INFINITY) - log; };
  for (int j = lane; j < a.asked; j += 64) {
    const LpAsked at = j == lane ? first : lp_asked<T>(a, row, j);
    a.lp[(size_t)row * a.asked + j] = at.in ? lp(at.x) : 0.f;
  }
  if (lane < a.k) {
    a.top_ids[(size_t)row * a.k + lane] = list.i;
    a.top_lp[(size_t)row * a.k + lane] = lp(list.v);
  }
}

// Workgroup (row, split): blocks split 4 W + wave, + 4 W S ...
template <class T, bool TOP>
__global__ __launch_bounds__(64 * kLpWaves) void k_logprobs(LpArgs a) {
  constexpr int kVec = 16 / sizeof(T);          // logits of 16 bytes
  constexpr int kParts = kLpBlock / 64 / kVec;  // 16-byte loads of a block
  __shared__ LpSlot slots[kLpWaves][64];
  __shared__ LpStats parts[kLpWaves];
  __shared__ uint32_t keys[TOP ? kLpKeys : 1][64 * kLpWaves];
  __shared__ int again;   // the keys do not tell
  const int row = blockIdx.x / a.S, split = blockIdx.x - row * a.S;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const T* xr = static_cast<const T*>(a.x) + (size_t)row * a.ld;
  // logits before the first 16-byte boundary and behind the last
  const int head = min(a.n, (int)((0u - (uint32_t)(uintptr_t)xr) % 16u / sizeof(T)));
  const u32x4* xv = reinterpret_cast<const u32x4*>(xr + head);
  const int vecs = (a.n - head) / kVec, tail = head + vecs * kVec;
  const int blocks = (vecs + 64 * kParts - 1) / (64 * kParts);
  const int b0 = split * kLpWaves + wave, step = kLpWaves * a.S;
  LpWave<TOP> w;
  // the eight that lane `of` has in block b: its 16-byte parts (past the row's, its last) --
  // there is one --, -Inf for those past the row's in its last block, its logits, their indices
  auto load = [&](u32x4 (&v)[kParts], int b, int of) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) v[p] = xv[min((b * kParts + p) * 64 + of, vecs - 1)];
  };
  auto end = [&](u32x4 (&v)[kParts], int b, int of) __attribute__((always_inline)) {
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      if ((b * kParts + p) * 64 + of >= vecs) v[p] = u32x4{kNone, kNone, kNone, kNone};
  };
  auto values = [&](float (&x)[8], const u32x4 (&v)[kParts]) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if constexpr (sizeof(T) == 4) {
          x[p * 4 + c] = __uint_as_float(v[p][c]);
        } else {
          x[2 * c] = bf16_bits_to_f32(v[p][c] & 0xffffu);
          x[2 * c + 1] = bf16_bits_to_f32(v[p][c] >> 16);
        }
  };
  auto index = [&](int b, int of, int e) { return head + ((b * kParts + e / kVec) * 64 + of) * kVec + e % kVec; };
  // use(x, block, number) for the wave's blocks, kLpAhead of them read at a time
  auto scan = [&](const auto& use) __attribute__((always_inline)) {
    for (int b = b0, number = 0; b < blocks; b += kLpAhead * step, number += kLpAhead) {
      u32x4 v[kLpAhead][kParts];
#pragma unroll
      for (int d = 0; d < kLpAhead; ++d) load(v[d], min(b + d * step, blocks - 1), lane);
#pragma unroll
      for (int d = 0; d < kLpAhead; ++d) {
        if (b + d * step >= blocks) break;
        float x[8];
        if (b + d * step == blocks - 1) end(v[d], b + d * step, lane);
        values(x, v[d]);
        use(x, b + d * step, (uint32_t)(number + d));
      }
    }
  };
  scan([&](const float (&x)[8], int, uint32_t number) __attribute__((always_inline)) {
    const float top = w.add(x, lane);
    if (TOP) w.remember(top, number);
  });
  const LpStats mine = w.stats(lane);
  if (lane == 0) parts[wave] = mine;
  if constexpr (TOP) {
#pragma unroll
    for (int l = 0; l < kLpKeys; ++l) keys[l][threadIdx.x] = w.key[l];
    __syncthreads();
    if (wave == 0) {
      uint32_t key[kLpKeys][kLpWaves], t = 0;
#pragma unroll
      for (int l = 0; l < kLpKeys; ++l)
#pragma unroll
        for (int o = 0; o < kLpWaves; ++o) key[l][o] = keys[l][64 * o + lane];
      // the order that the first keys of k lanes reach; at least that of a number
#pragma unroll
      for (int bit = 15; bit >= 0; --bit) {
        const uint32_t c = t | (1u << bit);
        int count = 0;
#pragma unroll
        for (int o = 0; o < kLpWaves; ++o) count += __popcll(__ballot(key[0][o] >= c << 16));
        if (count >= a.k) t = c;
      }
      t = max(t, kLpNone + 1) << 16;
      // the eights whose key reaches it, a lane each
      bool fits = a.few;
      int count = 0;
#pragma unroll
      for (int l = 0; l < kLpKeys; ++l)
#pragma unroll
        for (int o = 0; o < kLpWaves; ++o) {
          const unsigned long long some = __ballot(key[l][o] >= t);
          if (l == kLpKeys - 1 && some) fits = false;
          if (some) {
            const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
            if (key[l][o] >= t && at < 64)
              slots[0][at].i = (int)(((key[l][o] & 0xffffu) * (uint32_t)step + (uint32_t)(split * kLpWaves + o)) * 64u) + lane;
            count += __popcll(some);
          }
        }
      if (fits && count > 0 && count <= 64) {
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const bool has = lane < count;
        const int place = has ? slots[0][lane].i : 0, b = place >> 6, of = place & 63;   // block, its lane
        __builtin_amdgcn_wave_barrier();
        u32x4 v[kParts];
        float x[8];
        load(v, b, of);
        end(v, b, of);
        values(x, v);
        const float least = lp_least(t >> 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = has && x[e] >= least ? x[e] : -INFINITY;
        w.choose(x, [&](int e) { return index(b, of, e); }, a.k, lane, least, slots[0]);
      }
      if (lane == 0) again = !fits || count > 64;
    }
    __syncthreads();
    if (again)
      scan([&](const float (&x)[8], int b, uint32_t) __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
        if (__ballot(top > w.last))
          w.choose(x, [&](int e) { return index(b, lane, e); }, a.k, lane, w.first_least(top, a.k, lane), slots[wave]);
      });
    if (again) slots[wave][lane] = {w.list.v, w.list.i};
  }
  __syncthreads();
  if (wave) return;
  LpStats t = parts[0];
#pragma unroll
  for (int o = 1; o < kLpWaves; ++o) t = lp_join(t, parts[o]);
  if constexpr (TOP) {
    if (again) {
#pragma unroll
      for (int o = 1; o < kLpWaves; ++o) w.list.merge({slots[o][lane].v, slots[o][lane].i}, lane);
      w.close(a.k);
    }
  }
  if (split == 0) {   // the ends, less than 8 logits each
    w.m = t.m;
    w.s = lane == 0 ? t.s : 0.f;
    w.u = lane == 0 ? t.u : 0.f;
    w.own = lane == 0 && t.m > -INFINITY ? 1.f : 0.f;
#pragma unroll
    for (int end = 0; end < 2; ++end) {
      const int first = end ? tail : 0, count = end ? a.n - tail : head;
      if (count <= 0) continue;
      const float x[1] = {lane < count ? lp_logit(xr + first + lane) : -INFINITY};
      w.add(x, lane);
      if (TOP) w.choose(x, [&](int) { return first + lane; }, a.k, lane, -INFINITY, slots[0]);
    }
    t = w.stats(lane);
  }
  if (a.S == 1) {
    lp_write<T>(a, row, t, w.list, lp_asked<T>(a, row, lane), lane);
    return;
  }
  uint32_t* rec = a.part + (size_t)blockIdx.x * (4 + 2 * a.k);
  if (lane == 0) *reinterpret_cast<LpStats*>(rec) = t;
  if (lane < a.k) {
    rec[4 + lane] = __float_as_uint(w.list.v);
    rec[4 + a.k + lane] = (uint32_t)w.list.i;
  }
}

// A row's splits joined: wave w takes the splits w, w + 16, ..., then pairs of waves.
constexpr int kLpJoinWaves = 16, kLpMostSplits = 32;

template <class T>
__global__ __launch_bounds__(64 * kLpJoinWaves) void k_logprobs_join(LpArgs a) {
  __shared__ LpSlot slots[kLpJoinWaves][64];
  __shared__ LpStats parts[kLpJoinWaves];
  const int row = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  constexpr int kPer = kLpMostSplits / kLpJoinWaves;
  // all that the row needs is under way at once
  LpAsked first{};
  if (wave == 0) first = lp_asked<T>(a, row, lane);
  LpStats part[kPer];
  LpSlot slot[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int p = wave + kLpJoinWaves * j;
    const uint32_t* rec = a.part + ((size_t)row * a.S + min(p, a.S - 1)) * (4 + 2 * a.k);
    part[j] = *reinterpret_cast<const LpStats*>(rec);
    slot[j] = {-INFINITY, -1};
    if (lane < a.k) slot[j] = {__uint_as_float(rec[4 + lane]), (int)rec[4 + a.k + lane]};
  }
  LpStats t{-INFINITY, 0.f, 0.f};
  LpList list;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (wave + kLpJoinWaves * j >= a.S) break;
    t = lp_join(t, part[j]);
    if (a.k == 0) continue;
    if (j)
      list.merge({slot[j].v, slot[j].i}, lane);
    else
      list = {slot[j].v, slot[j].i};
  }
  for (int half = kLpJoinWaves / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      if (lane == 0) parts[wave] = t;
      slots[wave][lane] = {list.v, list.i};
    }
    __syncthreads();
    if (wave < half) {
      t = lp_join(t, parts[wave + half]);
      if (a.k) list.merge({slots[wave + half][lane].v, slots[wave + half][lane].i}, lane);
    }
  }
  if (wave == 0) lp_write<T>(a, row, t, list, first, lane);
}

// Workgroups a row is split over: one from 640 rows on; else some 1024 workgroups, of at least
// two blocks a wave, at most 32 a row. 256 / 400 rows of 248320 bf16 logits: 39 / 54 us, with
// some 512 workgroups 46 / 68, with 2048 42 / 54; 64 rows 21, 22 and 25; 1000 rows 103 whole, 112
// in two. One / 16 fp32 rows with 20 alternatives in 32 parts 13.3 / 15.8, in 16 13.9 / 15.3, in
// 64 14.0 / 17.2.
int lp_splits(int T, int n) {
  const long long blocks = ((long long)n + kLpBlock - 1) / kLpBlock;
  const long long most = blocks / (2 * kLpWaves);
  const long long want = T >= 640 ? 1 : (1024 + T - 1) / T;
  const long long s = want < most ? want : most;
  return s < 1 ? 1 : s > kLpMostSplits ? kLpMostSplits : (int)s;
}

size_t lp_bytes(int T, int n, int k) {
  const int S = lp_splits(T, n);
  return S == 1 ? 0 : (size_t)T * S * (4 + 2 * k) * 4;
}

template <class T>
int logprobs(float* lp, float* entropy, int32_t* top_ids, float* top_lp, const T* x, size_t ld,
             const int32_t* targets, int T_, int n, int asked, int k, qw4_workspace* ws, void* stream) {
  if (T_ < 0) return QW4_ERR_M;
  if (n < 1 || ld < (size_t)n || asked < 0 || k < 0 || k > kLpMaxTop) return QW4_ERR_SHAPE;
  if (T_ == 0) return QW4_OK;
  if (!x || (asked && (!lp || !targets)) || (k && (!top_ids || !top_lp))) return QW4_ERR_NULL;
  if ((uintptr_t)x % sizeof(T) || ((uintptr_t)lp | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_lp |
                                   (uintptr_t)targets) & 3)
    return QW4_ERR_ALIGN;
  const size_t need = lp_bytes(T_, n, k);
  LpArgs a{x, ld, targets, lp, entropy, top_lp, top_ids, n, asked, k, lp_splits(T_, n), 0, nullptr};
  a.few = (long long)n / kLpBlock < (1 << 24) && (long long)n / kLpBlock / (kLpWaves * a.S) < 65500;
  if (need) {
    if (!ws || !ws->buf || ws->bytes < need) return QW4_ERR_SCRATCH;
    if ((uintptr_t)ws->buf & 15) return QW4_ERR_ALIGN;
    a.part = static_cast<uint32_t*>(ws->buf);
  }
  hipStream_t s = (hipStream_t)stream;
  launch_rows_of(T_, 1 << 23, [&](int first, int rows) {
    LpArgs r = a;   // split rows are few: they go out in one run
    r.x = x + (size_t)first * ld;
    if (asked) {
      r.targets += (size_t)first * asked;
      r.lp += (size_t)first * asked;
    }
    if (entropy) r.entropy += first;
    if (k) {
      r.top_ids += (size_t)first * k;
      r.top_lp += (size_t)first * k;
    }
    if (k)
      k_logprobs<T, true><<<rows * r.S, 64 * kLpWaves, 0, s>>>(r);
    else
      k_logprobs<T, false><<<rows * r.S, 64 * kLpWaves, 0, s>>>(r);
    if (r.S > 1) k_logprobs_join<T><<<rows, 64 * kLpJoinWaves, 0, s>>>(r);
  });
  QW4_LAUNCH_CHECK();
  return QW4_OK;
}

}  // namespace
}  // namespace qw4

using namespace qw4;

extern "C" {

int qw4_logprobs(float* lp, float* entropy, int32_t* top_ids, float* top_lp, const uint16_t* logits, size_t ld,
                 const int32_t* targets, int T, int n, int asked, int top_k, qw4_workspace* ws, void* stream) {
  return logprobs<uint16_t>(lp, entropy, top_ids, top_lp, logits, ld, targets, T, n, asked, top_k, ws, stream);
}

int qw4_logprobs_f32(float* lp, float* entropy, int32_t* top_ids, float* top_lp, const float* logits, size_t ld,
                     const int32_t* targets, int T, int n, int asked, int top_k, qw4_workspace* ws, void* stream) {
  return logprobs<float>(lp, entropy, top_ids, top_lp, logits, ld, targets, T, n, asked, top_k, ws, stream);
}

size_t qw4_logprobs_workspace(int T, int n, int top_k) {
  return T < 1 || n < 1 || top_k < 0 || top_k > kLpMaxTop ? 0 : lp_bytes(T, n, top_k);
}

}  // extern "C"
