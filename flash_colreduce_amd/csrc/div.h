// Division by a number that a launch does not change.  Plain C++, so that it can be tested without a device.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define FCR_HOST_DEVICE __host__ __device__
#else
#define FCR_HOST_DEVICE
#endif

namespace fcr_paged {

// n / d for 0 <= n < 2^31 by one high product: m = floor(2^(31 + s) / d) + 1 with 2^(s - 1) < d <= 2^s, so that
// n m / 2^(31 + s) exceeds n / d by less than 2^-s <= 1 / d: the floor is the same.  m < 2^32.
struct Div {
  uint32_t mul, shift, d;
  void set(uint32_t by) {
    uint32_t s = 0;
    while ((1ull << s) < by) ++s;
    mul = by == 1 ? 0 : (uint32_t)((1ull << (31 + s)) / by + 1);
    shift = by == 1 ? 0 : s - 1;
    d = by;
  }
  FCR_HOST_DEVICE uint32_t of(uint32_t n) const {
    if (d == 1) return n;
    return (uint32_t)(((uint64_t)n * mul) >> 32) >> shift;
  }
};

}  // namespace fcr_paged
