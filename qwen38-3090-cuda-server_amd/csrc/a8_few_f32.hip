// The kernel for few rows, results in fp32.
#include "a8_few.h"

namespace qw4 {

bool a8_few_f32(const A8Args& a, int P, int U, bool small, hipStream_t st) {
  const FewArgs f{a, P, U};
  return small ? launch_few<A8_F32, 1>(f, st) : launch_few<A8_F32, 2>(f, st);
}

}  // namespace qw4
