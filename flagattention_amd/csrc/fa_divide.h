// Division of non-negative numbers by one that the host knows: a multiplication by its reciprocal
// and one correction (the compiler's own takes a dozen dependent steps and a trip through the
// vector unit, which a short kernel waits for).
#pragma once

#include "fa_common.h"

namespace fa {

struct Divisor {
  unsigned int by, inv;  // inv = floor((2^32 - 1) / by)
};

inline Divisor divisor(int by) {
  return Divisor{static_cast<unsigned int>(by), 0xFFFFFFFFu / static_cast<unsigned int>(by)};
}

// n < 2^31: n / by - n inv / 2^32 is below 1/2 + 1/2^32, so the estimate is at most one short.
__device__ inline int divide(int n, Divisor d) {
  const unsigned int x = static_cast<unsigned int>(n);
  const unsigned int q = __umulhi(x, d.inv);
  return static_cast<int>(x - q * d.by >= d.by ? q + 1 : q);
}

}  // namespace fa
