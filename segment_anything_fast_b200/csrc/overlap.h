// Do two strided operands share memory?  Host side: what an entry point writes may be an operand that its comment allows in
// place, or memory of its own; views of one buffer that lie between one another's rows are memory of their own too.
#pragma once

#include <stdint.h>

#include <utility>

namespace samb {

// n0 x n1 runs of `width` bytes, s0 and s1 bytes apart (strides not negative).
struct Runs {
  int64_t at, s0, n0, s1, n1, width;
};

inline Runs runs3(const void* at, int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t width) {
  Runs r{int64_t(reinterpret_cast<uintptr_t>(at)), s0, n0, s1, n1, width};
  if (at == nullptr || n0 <= 0 || n1 <= 0 || width <= 0) r.n0 = r.n1 = r.width = 0;
  // as few runs and axes as there are: axis 1 is the long one
  auto tidy = [&r]() {
    if (r.n1 == 1) {
      std::swap(r.s0, r.s1);
      std::swap(r.n0, r.n1);
    }
    if (r.n1 > 1 && r.s1 == r.width) {
      r.width *= r.n1;
      r.n1 = 1;
    }
  };
  tidy();
  if (r.n0 > 1 && r.n1 > 1 && r.s0 == r.s1 * r.n1) {
    r.n1 *= r.n0;
    r.n0 = 1;
  }
  tidy();
  if (r.n0 > r.n1) {
    std::swap(r.s0, r.s1);
    std::swap(r.n0, r.n1);
  }
  if (r.n0 <= 1) r.s0 = 0;
  if (r.n1 <= 1) r.s1 = 0;
  return r;
}
inline Runs rows_of(const void* at, int64_t pitch, int64_t n, int64_t width) { return runs3(at, 0, 1, pitch, n, width); }
inline Runs bytes_of(const void* at, int64_t n) { return runs3(at, 0, 1, 0, 1, n); }

inline int64_t end_of(const Runs& r) { return r.at + (r.n0 - 1) * r.s0 + (r.n1 - 1) * r.s1 + r.width; }

// Is d + j * s in (-below, above) for a j in [lo, hi]?  (s >= 0)
inline bool meets(int64_t d, int64_t s, int64_t lo, int64_t hi, int64_t below, int64_t above) {
  if (s == 0) return -below < d && d < above;
  auto floor_div = [s](int64_t v) { return v >= 0 ? v / s : -((-v + s - 1) / s); };
  const int64_t first = floor_div(-below - d) + 1, last = -floor_div(-(above - d)) - 1;
  return (first > lo ? first : lo) <= (last < hi ? last : hi);
}

inline bool share_memory(const Runs& a, const Runs& b) {
  if (a.width == 0 || b.width == 0 || end_of(a) <= b.at || end_of(b) <= a.at) return false;
  // run (i, j) of b against run (i', j') of a: their distance is b.at - a.at + i s0 + j s1 - i' s0' - j' s1', and they share
  // bytes where it lies in (-b.width, a.width)
  const int64_t d = b.at - a.at;
  if ((a.s0 == b.s0 || a.n0 == 1 || b.n0 == 1) && (a.s1 == b.s1 || a.n1 == 1 || b.n1 == 1)) {
    // only the differences of the indexes count
    const int64_t s0 = a.n0 > 1 ? a.s0 : b.s0, s1 = a.n1 > 1 ? a.s1 : b.s1;
    for (int64_t i = 1 - a.n0; i < b.n0; ++i)
      if (meets(d + i * s0, s1, 1 - a.n1, b.n1 - 1, b.width, a.width)) return true;
    return false;
  }
  // unlike pitches, one among the other's rows: seldom, and walked run by run
  for (int64_t i = 0; i < a.n0; ++i)
    for (int64_t j = 0; j < b.n0; ++j) {
      const int64_t e = d - i * a.s0 + j * b.s0;         // between their first runs
      if (a.n1 <= b.n1) {
        for (int64_t k = 0; k < a.n1; ++k)
          if (meets(e - k * a.s1, b.s1, 0, b.n1 - 1, b.width, a.width)) return true;
      } else {
        for (int64_t k = 0; k < b.n1; ++k)
          if (meets(-e - k * b.s1, a.s1, 0, a.n1 - 1, a.width, b.width)) return true;
      }
    }
  return false;
}

}  // namespace samb
