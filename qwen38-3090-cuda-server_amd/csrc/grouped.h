// Shared by the products grouped by expert: arguments, and how a workgroup finds its
// work from the plan's offsets.
#pragma once
#include <hip/hip_runtime.h>

#include "epilogue.h"
#include "w4a16_common.h"

namespace qw4 {

constexpr int kMaxExperts = 1024;

struct GroupedArgs {
  const uint32_t* qw;
  const uint16_t* sc;
  const uint16_t* zr;
  const uint16_t* x;
  uint16_t* y;
  const int32_t* offsets;   // [E + 1]
  const int32_t* tokens;    // row of x at each position
  Epilogue epi;             // bias and up of an expert's weight rows; no residual
  int E, n, K, G;           // n weight rows an expert
  int R;                    // positions (rows of y)
  uint32_t x_bytes;         // of a gathered x
  int ld;                   // columns of y
  int tiles_n, P;           // column tiles of an expert, workgroups
  const int *rexp, *cexp;   // fp16 operands: exponents of x's rows and of the weight rows
};

// Expert e's positions. Offsets that are no plan's (negative, falling, past R) give
// fewer or no rows, never one outside y.
__device__ __forceinline__ void expert_rows(const GroupedArgs& a, int e, int& lo, int& hi) {
  lo = min(max(a.offsets[e], 0), a.R);
  hi = min(max(a.offsets[e + 1], lo), a.R);
}

// Running sums over the experts of N counts each, count(rows, which): start[which
// (kMaxExperts + 1) + e] = those of the experts before e, all[which] = the total. For a
// workgroup of THREADS; wsum [THREADS / 64 N].
template <int THREADS, int N, class Count>
__device__ __forceinline__ void expert_starts(const GroupedArgs& a, int* start, int* wsum, int (&all)[N],
                                              const Count& count) {
  constexpr int kPer = kMaxExperts / THREADS;   // experts of a thread
  constexpr int kWaves = THREADS / 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int n[N][kPer], run[N];
#pragma unroll
  for (int w = 0; w < N; ++w) run[w] = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = kPer * t + i;
    int lo = 0, hi = 0;
    if (e < a.E) expert_rows(a, e, lo, hi);
#pragma unroll
    for (int w = 0; w < N; ++w) {
      n[w][i] = count(hi - lo, w);
      run[w] += n[w][i];
    }
  }
  int before[N];
#pragma unroll
  for (int w = 0; w < N; ++w) {
    before[w] = -run[w];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(run[w], off, 64);
      if (lane >= off) run[w] += v;
    }
    before[w] += run[w];
    if (lane == 63) wsum[w * kWaves + wave] = run[w];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < N; ++w) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      before[w] += i < wave ? wsum[w * kWaves + i] : 0;
      sum += wsum[w * kWaves + i];
    }
    all[w] = __builtin_amdgcn_readfirstlane(sum);
    int* const s = start + w * (kMaxExperts + 1);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      s[kPer * t + i] = before[w];
      before[w] += n[w][i];
    }
    if (t == THREADS - 1) s[kMaxExperts] = before[w];
  }
  __syncthreads();
}

// The last expert whose first tile is at or before t (experts without tiles start where
// the next one does, so it has some).
__device__ __forceinline__ int expert_of(const int* start, int E, int tiles_n, int t) {
  int lo = 0, hi = E;   // start[lo] tiles_n <= t < start[hi] tiles_n
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] * tiles_n <= t)
      lo = mid;
    else
      hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The kernel for these arguments (qw4_tune_grouped's numbers; 3 for tiles of 128 or 256),
// of those alone that use the weights exactly if `exact` is set and they apply.
int grouped_form(const GroupedArgs& a, bool glu, int cus, bool exact);
// Forms 1 and 2 (grouped_rows.hip): launches it and returns true, or returns false where it
// is another or does not apply.
bool grouped_rows_launch(GroupedArgs& a, bool glu, int cus, int form, hipStream_t s);

}  // namespace qw4
