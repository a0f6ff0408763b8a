// The kernel for few rows with an epilogue (not gated).
#include "a8_few.h"

namespace qw4 {

bool a8_few_epi(const A8Args& a, int P, int U, bool small, hipStream_t st) {
  const FewArgs f{a, P, U};
  return small ? launch_few<A8_EPI, 1>(f, st) : launch_few<A8_EPI, 2>(f, st);
}

}  // namespace qw4
