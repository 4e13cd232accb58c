// The tanh of capped scores (wechat-tfcc_amd/csrc/score_tanh.hpp), the code that the kernels run, against 64 bits.  No GPU.
#include <cmath>
#include <cstdio>
#include <limits>

#include "score_tanh.hpp"

using namespace tfcc_rocm;

static int failures = 0;
#define EXPECT(cond)                                         \
  do {                                                       \
    if (!(cond)) {                                           \
      ++failures;                                            \
      std::printf("FAIL line %d: %s\n", __LINE__, #cond);    \
    }                                                        \
  } while (0)

static float far_of(float x) {
  return tanh_far(x, [](float v) { return std::exp2(v); }, [](float v) { return 1.0f / v; });
}

int main() {
  const double unit = std::ldexp(1.0, -24);  // half a step of float32, relative
  // Near: 2^-27 of the polynomial, half a step of the last sum and what its second part brings, which is 0.11 of the result at most: the rounding of x * y, of P and of y in it, 4 half steps
  // of that part.  Half a step is 2^-24 of numbers at the low end of their power of two.
  double worst = 0;
  for (unsigned bits = 0x00800000u; bits < 0x3f0ccccdu; bits += 997) {  // the smallest normal number to 0.55
    float x;
    static_assert(sizeof x == sizeof bits, "");
    __builtin_memcpy(&x, &bits, 4);
    const double want = std::tanh((double)x), off = std::fabs((double)tanh_near(x) - want) / want;
    worst = off > worst ? off : worst;
    EXPECT(tanh_near(-x) == -tanh_near(x));
  }
  EXPECT(worst <= (1 + 4 * 0.11 + 0.125) * unit);
  std::printf("below the border: %.3f half steps\n", worst / unit);
  EXPECT(tanh_near(0.0f) == 0.0f);
  // Far: 1 - u, u = 2 / (e + 1) of 0.5 at most of a result of 0.5 at least.  The exponent is off by half a step of 2 log2(e) x and of its factor, 2 ln(2) x half steps of the power; the power, the sum
  // and the inverse half a step to a step each: u is off by 2.8 x + 4 half steps of itself, x u tanh(x)^-1 being 0.55 x 1 at the border and less above.
  worst = 0;
  for (float x = kTanhNear; x < 50; x = x * 1.00001f) {
    const double want = std::tanh((double)x), u = 1 - want, off = std::fabs((double)far_of(x) - want) / want;
    EXPECT(off <= (1 + (2.8 * x + 5) * u / want) * unit);
    worst = off > worst ? off : worst;
    const double below = (double)far_of(-x) + want;
    EXPECT(std::fabs(below) / want <= (1 + (2.8 * x + 5) * (1 + want) / want) * unit);
  }
  std::printf("above it: %.3f half steps\n", worst / unit);
  const float infinity = std::numeric_limits<float>::infinity();
  EXPECT(far_of(infinity) == 1.0f && far_of(-infinity) == -1.0f && far_of(3.4e38f) == 1.0f && far_of(-3.4e38f) == -1.0f);
  EXPECT(std::isnan(far_of(NAN)) && std::isnan(tanh_near(NAN)));
  if (failures == 0) std::printf("score tanh: all passed\n");
  return failures != 0;
}
