// Host run of how the 8-bit cache's kernels hold a stored scale (csrc/kv8.h): itself in the range,
// between 2^-50 and 2^51 whatever the bits are.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../tiledattention_b200/csrc/kv8.h"

using namespace ta::kv8;

int main() {
  int checks = 0;
  const float least = std::ldexp(1.f, kScaleExpMin), most = std::ldexp(1.f, kScaleExpMax + 1);
  for (uint32_t sign : {0u, 1u})
    for (uint32_t e = 0; e < 256; ++e)
      for (uint32_t m = 0; m < (1u << 23); m = m < 600 || m >= (1u << 23) - 600 ? m + 1 : m + 499) {
        const uint32_t bits = sign << 31 | e << 23 | m, held = held_scale(bits);
        float f, h;
        std::memcpy(&f, &bits, 4);
        std::memcpy(&h, &held, 4);
        ++checks;
        const bool inside = std::fabs(f) >= least && std::fabs(f) < most;
        if (!(h >= least && h < most) || (inside && h != std::fabs(f)) ||
            (held & 0x7fffffu) != m || stored_exponent(held) != stored_exponent(bits)) {
          std::printf("FAIL %08x %08x\n", bits, held);
          return 1;
        }
      }
  std::printf("ok %d\n", checks);
  return 0;
}
