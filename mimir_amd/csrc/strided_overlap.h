// Whether strided regions of memory share a byte, exactly (host code).
//
// Two views of one tensor may lie in the same range of addresses without sharing anything: the query
// and key heads of a fused projection, heads dealt alternately, heads in front of tokens.  They share a
// byte where the difference of two of their addresses, a sum of coefficients times
// strides, is zero.  The coefficient of the largest stride is bounded by what the smaller ones can make
// up for, so for nested strides (each at least the span of the smaller ones) one or two values are
// left to look at for each.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdlib>

namespace mimir {

// Runs of `run` bytes at base + sum_i c_i stride[i], 0 <= c_i < size[i]; strides in bytes.
struct Region {
  static constexpr int kDims = 3;
  const void* base;
  int64_t run, size[kDims], stride[kDims];
};

namespace overlap {

struct Term {
  int64_t stride, lo, hi;  // stride times a coefficient in [lo, hi]
};
struct Terms {
  Term t[2 * Region::kDims + 1];
  int n = 0;
  void add(int64_t stride, int64_t lo, int64_t hi) {
    if (lo == hi || stride == 0) return;  // (lo <= 0 <= hi)
    if (stride < 0) {
      stride = -stride;
      std::swap(lo, hi);
      lo = -lo, hi = -hi;
    }
    for (int i = 0; i < n; ++i)
      if (t[i].stride == stride) {
        t[i].lo += lo, t[i].hi += hi;
        return;
      }
    t[n++] = {stride, lo, hi};
  }
  void sort() {
    std::sort(t, t + n, [](const Term& a, const Term& b) { return a.stride > b.stride; });
  }
};

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0

// Whether at + sum_i c_i stride_i = 0 for some coefficients (`other`: that are not all zero).  After `tries`
// steps, far more than nested strides take, it says so without knowing.
inline bool reaches_zero(const Term* t, int n, int64_t at, bool other, int& tries) {
  if (n == 0) return at == 0 && !other;
  int64_t lo = at, hi = at;  // with what the smaller strides can add
  for (int i = 1; i < n; ++i) lo += t[i].lo * t[i].stride, hi += t[i].hi * t[i].stride;
  const int64_t first = std::max(t->lo, -floor_div(hi, t->stride)), last = std::min(t->hi, floor_div(-lo, t->stride));
  for (int64_t c = first; c <= last; ++c)
    if (--tries < 0 || reaches_zero(t + 1, n - 1, at + c * t->stride, other && c == 0, tries)) return true;
  return false;
}
constexpr int kTries = 4096;

}  // namespace overlap

// The bytes of the region's range of addresses, and where it starts.
inline uintptr_t range(const Region& a, uintptr_t& start) {
  int64_t below = 0, above = a.run;
  for (int i = 0; i < Region::kDims; ++i) (a.stride[i] < 0 ? below : above) += (a.size[i] - 1) * a.stride[i];
  start = (uintptr_t)a.base + below;
  return above - below;
}

inline bool empty(const Region& a) { return a.run <= 0 || std::min({a.size[0], a.size[1], a.size[2]}) <= 0; }

// Whether two runs of the region share a byte.
inline bool overlaps_itself(const Region& a) {
  if (empty(a)) return false;
  // nearly always: each stride at least the span of the smaller ones
  int order[Region::kDims] = {0, 1, 2};
  auto step = [&](int i) { return a.size[i] == 1 ? 0 : std::abs(a.stride[i]); };
  for (int pair : {0, 1, 0})
    if (step(order[pair]) > step(order[pair + 1])) std::swap(order[pair], order[pair + 1]);
  bool nested = true;
  int64_t span = a.run;
  for (int i : order) {
    if (a.size[i] == 1) continue;
    nested = nested && step(i) >= span;
    span += (a.size[i] - 1) * step(i);
  }
  if (nested) return false;
  overlap::Terms s;
  for (int i = 0; i < Region::kDims; ++i) {
    if (a.size[i] > 1 && a.stride[i] == 0) return true;
    s.add(a.stride[i], 1 - a.size[i], a.size[i] - 1);
  }
  // dims of one stride were added up: their own coefficients cancel
  int dims = 0;
  for (int i = 0; i < Region::kDims; ++i) dims += a.size[i] > 1;
  if (s.n < dims) return true;
  s.add(1, 1 - a.run, a.run - 1);
  s.sort();
  int tries = overlap::kTries;
  return overlap::reaches_zero(s.t, s.n, 0, true, tries);
}

// Whether the regions share a byte.
inline bool overlap_each_other(const Region& a, const Region& b) {
  if (empty(a) || empty(b)) return false;
  uintptr_t a0, b0;
  const uintptr_t na = range(a, a0), nb = range(b, b0);
  if (a0 - b0 >= nb && b0 - a0 >= na) return false;
  overlap::Terms s;
  for (int i = 0; i < Region::kDims; ++i) {
    s.add(a.stride[i], 0, a.size[i] - 1);
    s.add(b.stride[i], 1 - b.size[i], 0);
  }
  s.add(1, 1 - b.run, a.run - 1);
  s.sort();
  int tries = overlap::kTries;
  return overlap::reaches_zero(s.t, s.n, (int64_t)((uintptr_t)a.base - (uintptr_t)b.base), false, tries);
}

}  // namespace mimir
