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
};

// Expert e's positions. Offsets that are no plan's (negative, falling, past R) give
// fewer or no rows, never one outside y.
__device__ __forceinline__ void expert_rows(const GroupedArgs& a, int e, int& lo, int& hi) {
  lo = min(max(a.offsets[e], 0), a.R);
  hi = min(max(a.offsets[e + 1], lo), a.R);
}

// Blocks of ROWS positions: start[e] = those of the experts before e, returned: all.
// For a workgroup of THREADS, start [kMaxExperts + 1] and wsum [THREADS / 64] in LDS.
template <int ROWS, int THREADS>
__device__ __forceinline__ int block_starts(const GroupedArgs& a, int* start, int* wsum) {
  constexpr int kPer = kMaxExperts / THREADS;   // experts of a thread
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int n[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = kPer * t + i;
    n[i] = 0;
    if (e < a.E) {
      int lo, hi;
      expert_rows(a, e, lo, hi);
      n[i] = (hi - lo + ROWS - 1) / ROWS;
    }
    sum += n[i];
  }
  int run = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(run, off, 64);
    if (lane >= off) run += v;
  }
  if (lane == 63) wsum[wave] = run;
  __syncthreads();
  int before = run - sum, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    before += w < wave ? wsum[w] : 0;
    all += wsum[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (kPer * t + i <= a.E) start[kPer * t + i] = before;
    before += n[i];
  }
  if (t == THREADS - 1 && a.E == kMaxExperts) start[kMaxExperts] = before;
  __syncthreads();
  return all;
}

// The last expert whose first tile is at or before t (experts without rows start where
// the next one does, so it has rows).
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

// Few rows an expert (grouped_rows.hip): launches it and returns true, or returns false
// where it does not apply.
bool grouped_rows_launch(GroupedArgs& a, bool glu, int cus, hipStream_t s);

}  // namespace qw4
