// The mean of a sum that is a whole multiple of the width is exact, and of any sum off by at most half a step and a
// hair.  Arguments: first width, last width.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "zp_rowwise.cuh"

int main(int, char **argv) {
  std::mt19937 rng(1);
  std::uniform_real_distribution<float> any(-4096.f, 4096.f);
  for (int width = std::atoi(argv[1]); width <= std::atoi(argv[2]); ++width) {
    const ZpOver over = zp_over(width);
    for (int i = 0; i < 64; ++i) {
      // a mean whose product with the width has 24 bits at most
      int bits = 24;
      while (width >> (24 - bits)) --bits;
      float mean = std::ldexp(std::floor(std::ldexp(any(rng) / 4096.f, bits)), (int)(rng() % 40) - 20 - bits);
      const float sum = mean * (float)width;
      if ((double)sum != (double)mean * width) return std::printf("%d: the sum is not exact\n", width), 1;
      if (over.of(sum) != mean) return std::printf("%d: %.9g instead of %.9g\n", width, over.of(sum), mean), 1;
      const float s = any(rng), got = over.of(s);
      const double want = (double)s / width, step = std::ldexp(1.0, std::ilogb(want) - 23);
      if (!(std::abs(got - want) <= step * (0.5 + 1e-6))) return std::printf("%d: off by %g steps\n", width, std::abs(got - want) / step), 1;
    }
  }
  if (zp_over(1000).of(0.f) != 0.f) return std::puts("zero"), 1;
  std::puts("ok");
}
