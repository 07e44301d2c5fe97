// Whether strided pools share memory (host code): a pool holds rows of `row` bytes at the sums of
// one multiple of each axis's stride.
#pragma once

#include <stdint.h>

namespace pools {

struct Axis {
  int64_t stride, count;  // bytes, entries
};

// Some difference of indices within the axes (the widest stride first) lies less than a row from
// `delta`.  An axis's multiple is one of the two next to it where the axes behind it stay below
// its stride.
inline bool meets(int64_t delta, const Axis* axes, int n, int64_t row) {
  if (delta < 0) delta = -delta;
  if (n == 0) return delta < row;
  const int64_t q = delta / axes[0].stride;
  for (int64_t k = q; k <= q + 1; ++k)
    if (k < axes[0].count && meets(delta - k * axes[0].stride, axes + 1, n - 1, row)) return true;
  return false;
}

// Rows of one pool share bytes, or rows of two pools of the layout that lie `delta` bytes apart.
inline bool overlap(int64_t delta, const Axis (&layout)[3], int64_t row) {
  Axis axes[3];
  int n = 0;
  for (Axis a : layout) {
    if (a.stride < 0) a.stride = -a.stride;
    if (a.count < 2) continue;
    if (a.stride < row) return true;
    int at = n++;
    for (; at > 0 && axes[at - 1].stride < a.stride; --at) axes[at] = axes[at - 1];
    axes[at] = a;
  }
  int64_t inside = row;  // bytes that the axes behind i span
  for (int i = n - 1; i >= 0; --i) {
    for (int64_t k = 1; k < axes[i].count && k * axes[i].stride < inside; ++k)
      if (meets(k * axes[i].stride, axes + i + 1, n - i - 1, row)) return true;
    inside += (axes[i].count - 1) * axes[i].stride;
  }
  return meets(delta, axes, n, row);
}

// Rows [i, a head of `heads`] and [j, a head of `others`] of `dim` elements, i and j below `rows`, in
// tensors of the same row and head strides (not negative) that begin `delta` elements apart, share one.
inline bool rows_meet(int64_t delta, int64_t row, int64_t head, int64_t rows, int64_t heads, int64_t others,
                      int64_t dim) {
  if (rows < 2) row = 0;
  for (int64_t n = 1 - others; n < heads; ++n) {
    const int64_t left = delta - n * head;
    // (row differences next to the one that leaves nothing, or the last of them)
    int64_t q = row ? left / row : 0;
    q = q < -rows ? -rows : q > rows ? rows : q;
    for (int64_t r = q - 1; r <= q + 1; ++r) {
      const int64_t away = left - r * row;
      if (r > -rows && r < rows && away < dim && -away < dim) return true;
    }
  }
  return false;
}

}  // namespace pools
