// Which calls the kernel for few rows (a8_few.h) takes, and its gated forms; the others are
// compiled beside it.
#include "a8_few.h"

namespace qw4 {

// Launches the rows of `a` where this kernel takes them.
bool a8_few(int out, const A8Args& a, int cus, hipStream_t st) {
  if (a.M > 64) return false;
  if ((size_t)a.N * a.K / 2 >= (1ull << 32) || (size_t)a.M * a.K >= (1ull << 32)) return false;   // 32-bit offsets
  const int tiles = a.ld / kTileN;
  // 16-row units while they leave no workgroup two (4096 x 5120, one / 9 rows 5.0 / 5.8 us, in
  // units of 32 rows 5.5 / 6.8; 7168 x 5120 7.2 / 7.9 and 6.0 / 7.1)
  const bool small = out == A8_GLU ? a.M > 32 : 4 * tiles <= cus;
  const int S = small ? 1 : 2;
  const int U = tiles * 4 / S;
  // as few workgroups as give none of them another unit
  const int most = (U + cus - 1) / cus;
  const int P = (U + most - 1) / most;
  if (out == A8_GLU)
    return small ? launch_few<A8_GLU, 1>(FewArgs{a, P, U}, st) : launch_few<A8_GLU, 2>(FewArgs{a, P, U}, st);
  return out == A8_F32 ? a8_few_f32(a, P, U, small, st) : a8_few_epi(a, P, U, small, st);
}

}  // namespace qw4
