// Whether rows of memory that a kernel writes lie apart.  Plain C++, so that it can be tested without a device.
#pragma once

#include <stdint.h>

namespace fcr_paged {

struct Dimension {
  int64_t size, stride;
};

// Rows of `row` elements in dimensions of any order.  Apart, if every dimension, by rising strides, steps over all that those before it span:
// true of every layout that a tensor and its slices and transposes have.  (Strides are in [0, 2^40), sizes below 2^31.)
inline bool rows_apart(int64_t row, const Dimension* of, int n) {
  Dimension d[4];
  int m = 0;
  for (int i = 0; i < n; ++i) {
    if (of[i].size <= 1) continue;               // (its stride is never used)
    int j = m++;
    for (; j > 0 && d[j - 1].stride > of[i].stride; --j) d[j] = d[j - 1];
    d[j] = of[i];
  }
  __int128 span = row;
  for (int i = 0; i < m; ++i) {
    if (d[i].stride < span) return false;
    span += (__int128)(d[i].size - 1) * d[i].stride;
  }
  return true;
}

// Two sets of such rows, at x and y (byte addresses of elements of `bytes` bytes).  Of two that are laid out alike the distance is one more
// dimension; otherwise only a common start is known to be wrong.
inline bool rows_apart(int64_t row, const Dimension* x_dims, uintptr_t x, const Dimension* y_dims, uintptr_t y, int n, int bytes) {
  if (!rows_apart(row, x_dims, n) || !rows_apart(row, y_dims, n) || x == y) return false;
  Dimension all[4];
  for (int i = 0; i < n; ++i) {
    if (x_dims[i].size > 1 && x_dims[i].stride != y_dims[i].stride) return true;
    all[i] = x_dims[i];
  }
  all[n] = Dimension{2, (int64_t)((x > y ? x - y : y - x) / (uintptr_t)bytes)};
  return rows_apart(row, all, n + 1);
}

}  // namespace fcr_paged
