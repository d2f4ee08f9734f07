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

// Arrays of rows of `row` elements, none of which shares memory with another of its array; the second array starts `distance` elements
// behind the first.  Exact where both have the same strides.  Otherwise true where the rows' places between their strides' common divisor
// meet, which is to be taken as "it may be".
inline bool share(std::vector<Axis> axes, int64_t row, int64_t distance) {
  for (const Axis& x : axes)
    if (x.size == 0) return false;
  if (row == 0) return false;
  axes.erase(std::remove_if(axes.begin(), axes.end(), [](const Axis& x) { return x.size == 1; }), axes.end());
  if (distance >= span(axes, row, [](const Axis& x) { return x.a; }) || -distance >= span(axes, row, [](const Axis& x) { return x.b; })) return false;
  if (std::all_of(axes.begin(), axes.end(), [](const Axis& x) { return x.a == x.b; })) {
    std::sort(axes.begin(), axes.end(), [](const Axis& x, const Axis& y) { return x.a > y.a; });
    return reaches(axes, 0, row, distance);
  }
  int64_t every = 0;
  for (const Axis& x : axes) every = std::gcd(every, std::gcd(x.a, x.b));
  const int64_t at = (distance % every + every) % every;
  return at < row || every - at < row;
}

}  // namespace msd_overlap

#endif  // MSD_OVERLAP_H
