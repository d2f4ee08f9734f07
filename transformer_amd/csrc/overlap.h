// Whether two strided arrays of one shape share memory (host code).
#ifndef MSD_OVERLAP_H
#define MSD_OVERLAP_H

#include <stdint.h>
#include <stdlib.h>

#include <algorithm>
#include <numeric>
#include <vector>

namespace msd_overlap {

struct Axis {
  int64_t size, a, b;   // strides in the two arrays, in elements
};

// Places of an array whose element 0 is at 0: one past the last
template <class F>
int64_t span(const std::vector<Axis>& axes, int64_t row, F stride) {
  int64_t end = row;
  for (const Axis& x : axes) end += (x.size - 1) * stride(x);
  return end;
}

// One stride for both on every axis from i on, the largest first, each at least the places of those behind it: the distance is
// sum_i d_i stride_i + d with |d_i| < size_i and |d| < row for two elements that are one.  What the axes behind i make up is less than stride_i, so
// d_i is one of two.
inline bool reaches(const std::vector<Axis>& axes, size_t i, int64_t row, int64_t distance) {
  if (i == axes.size()) return llabs(distance) < row;
  const int64_t s = axes[i].a, low = distance / s - (distance % s < 0);
  for (const int64_t d : {low, low + 1})
    if (llabs(d) < axes[i].size && reaches(axes, i + 1, row, distance - d * s)) return true;
  return false;
}

// The same with axes of different strides in front, whose places are tried one by one
inline bool reaches(const std::vector<Axis>& apart, size_t i, const std::vector<Axis>& axes, int64_t row, int64_t distance) {
  if (i == apart.size()) return reaches(axes, 0, row, distance);
  for (int64_t a = 0; a < apart[i].size; ++a)
    for (int64_t b = 0; b < apart[i].size; ++b)
      if (reaches(apart, i + 1, axes, row, distance - a * apart[i].a + b * apart[i].b)) return true;
  return false;
}

// Arrays of rows of `row` elements, none of which shares memory with another of its array; the second array starts `distance` elements
// behind the first.  Exact, unless axes of different strides (heads, say, that are dealt out in two ways) have more than `most` pairs of places:
// then true where the rows' places between the strides' common divisor meet, which is to be taken as "it may be".
inline bool share(std::vector<Axis> axes, int64_t row, int64_t distance, int64_t most = 1 << 14) {
  for (const Axis& x : axes)
    if (x.size == 0) return false;
  if (row == 0) return false;
  axes.erase(std::remove_if(axes.begin(), axes.end(), [](const Axis& x) { return x.size == 1; }), axes.end());
  if (distance >= span(axes, row, [](const Axis& x) { return x.a; }) || -distance >= span(axes, row, [](const Axis& x) { return x.b; })) return false;
  std::sort(axes.begin(), axes.end(), [](const Axis& x, const Axis& y) { return x.a > y.a; });
  std::vector<Axis> apart;
  int64_t pairs = 1, every = 0;
  for (const Axis& x : axes) {
    every = std::gcd(every, std::gcd(x.a, x.b));
    if (x.a == x.b) continue;
    apart.push_back(x);
    pairs = pairs > most / x.size / x.size ? most + 1 : pairs * x.size * x.size;
  }
  if (pairs > most && !apart.empty()) {
    const int64_t at = (distance % every + every) % every;
    return at < row || every - at < row;
  }
  axes.erase(std::remove_if(axes.begin(), axes.end(), [](const Axis& x) { return x.a != x.b; }), axes.end());
  return reaches(apart, 0, axes, row, distance);
}

}  // namespace msd_overlap

#endif  // MSD_OVERLAP_H
