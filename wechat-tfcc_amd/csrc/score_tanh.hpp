// tanh of scores over their cap, to about float32's last place, of the result and not of 1: below kTanhNear x + x^3 P(x^2) with P of degree 4 fitted for the smallest relative error (its
// coefficients, rounded to float32, leave 2^-27.0 at the border and less below), above, 1 - 2 / (2^(2 log2(e) x) + 1).
//
// Plain functions of numbers, compiled for the device by the kernels and for the host by the test that measures them.
#pragma once

#include <math.h>

#if defined(__HIPCC__)
#define TFCC_TANH_HD __host__ __device__ __forceinline__
#else
#define TFCC_TANH_HD inline
#endif

namespace tfcc_rocm {

constexpr float kTanhNear = 0.55f;

TFCC_TANH_HD float tanh_near(float x) {
  const float y = x * x;
  float r = -0.00627424f;
  r = fmaf(r, y, 0.02107168f);
  r = fmaf(r, y, -0.05385231f);
  r = fmaf(r, y, 0.13332586f);
  r = fmaf(r, y, -0.33333318f);
  return fmaf(x * y, r, x);
}

// exp2 and inverse: 2^v and 1 / v, to about a unit in the last place.  An infinity gives 1 under its sign.
template <class Exp2, class Inverse>
TFCC_TANH_HD float tanh_far(float x, Exp2 exp2_of, Inverse inverse_of) {
  return fmaf(-2.0f, inverse_of(exp2_of(x * 2.88539008177792681f) + 1.0f), 1.0f);
}

}  // namespace tfcc_rocm
