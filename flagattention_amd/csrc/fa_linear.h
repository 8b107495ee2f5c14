// What the kernels of linear attention share: powers of the decay, the checks of their arguments.
#pragma once

#include "fa_common.h"
#include "flagattention_amd_linear.h"

namespace fa {

// e^(a n), 1 for n = 0 whatever a is (also -inf, a decay to nothing).
__device__ inline float decay(float a, int n) {
  return n == 0 ? 1.f : expf(a * static_cast<float>(n));
}
// S times e^(a n).  A slow decay is taken as S + S (e^(a n) - 1): next to 1 e^(a n) itself has lost bits,
// 2^-25 of S a step and always the same way (1e-4 after 4,000 steps).  A fast one is a product: there
// the difference would lose them.
struct Fall {
  float by, keep;  // S keep + S by, keep is 1 or 0
};
__device__ inline Fall fall_of(float a, int n) {
  const float x = a * static_cast<float>(n);
  const bool slow = x > -0.5f;
  return Fall{n == 0 ? 0.f : slow ? expm1f(x) : expf(x), slow || n == 0 ? 1.f : 0.f};
}
// more + S e^(a n): rounded at S's size once.
__device__ inline float add_fallen(float s, Fall fall, float more) {
  return __builtin_fmaf(s, fall.keep, __builtin_fmaf(s, fall.by, more));
}

int check_linear_shape(const fa_linear_args& a);
int check_linear(const fa_linear_args& a);

}  // namespace fa
