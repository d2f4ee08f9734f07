// Compares transformer_amd/csrc/overlap.h with lists of places, over small arrays of all kinds: they have to agree, and where the strides
// differ and no places are tried one by one, arrays must not be called apart where they meet.  Prints how many were compared of each kind
// and answer.
#include <cstdio>
#include <random>
#include <set>

#include "../transformer_amd/csrc/overlap.h"

using msd_overlap::Axis;

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int a, int b) { return std::uniform_int_distribution<int>(a, b)(rng); };
  long same[2] = {}, other[2] = {}, refused = 0;
  for (int n = 0; n < 400000; ++n) {
    const int row = pick(1, 4), dims = pick(0, 3);
    std::vector<Axis> axes(dims);
    // strides from the innermost out, with room between; those of the second array the same, or of another order of the axes
    const bool one = pick(0, 2) > 0;
    int64_t a = row + pick(0, 3), b = row + pick(0, 3);
    for (Axis& x : axes) {
      x = {pick(1, 4), a, one ? a : b};
      a = a * x.size + pick(0, 3);
      b = b * x.size + pick(0, 3);
    }
    std::shuffle(axes.begin(), axes.end(), rng);
    bool equal = true;
    for (const Axis& x : axes) equal &= x.size == 1 || x.a == x.b;
    const int64_t distance = pick(-150, 150);
    auto places = [&](bool second) {
      std::vector<int64_t> at{second ? distance : 0};
      for (const Axis& x : axes) {
        std::vector<int64_t> next;
        for (const int64_t p : at)
          for (int64_t i = 0; i < x.size; ++i) next.push_back(p + i * (second ? x.b : x.a));
        at = next;
      }
      std::set<int64_t> all;
      for (const int64_t p : at)
        for (int i = 0; i < row; ++i) all.insert(p + i);
      return all;
    };
    const auto p = places(false), q = places(true);
    bool meet = false;
    for (const int64_t x : p) meet |= q.count(x) > 0;
    if (meet != msd_overlap::share(axes, row, distance)) return std::printf("not exact\n"), 1;
    const bool said = msd_overlap::share(axes, row, distance, 0);
    if (meet && !said) return std::printf("missed\n"), 1;
    if (equal && meet != said) return std::printf("not exact\n"), 1;
    ++(equal ? same : other)[meet];
    refused += said && !meet;
  }
  // empty arrays share nothing
  if (msd_overlap::share({{0, 8, 8}}, 4, 0) || msd_overlap::share({{2, 8, 8}}, 0, 0)) return std::printf("empty\n"), 1;
  std::printf("same %ld %ld other %ld %ld refused %ld\n", same[0], same[1], other[0], other[1], refused);
}
