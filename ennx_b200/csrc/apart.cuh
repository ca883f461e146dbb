// apart.cuh -- do the operands of a call share memory?  Host code without CUDA.
#pragma once

#include <stdint.h>

namespace ennx {

// Memory that a call reads or writes: runs of `run` bytes, `count[d]` of them
// `stride[d]` bytes apart (not negative) in each of up to three dimensions.
struct Memory {
  const void* base = nullptr;
  int64_t run = 0, count[3] = {1, 1, 1}, stride[3] = {};
  static Memory bytes(const void* p, int64_t n) { return {p, n, {1, 1, 1}, {}}; }
  static Memory rows(const void* p, int64_t n, int64_t stride, int64_t run) { return {p, run, {n, 1, 1}, {stride, 0, 0}}; }
};

namespace apart {
typedef __int128 wide;
// n * stride for an n in [lo, hi]
struct Term {
  wide stride, lo, hi;
};
// Is there a sum of one value per term in (low, high)?  Terms are sorted, the
// largest stride first; of each only the values that the smaller ones can still
// bring there are tried.
inline bool some_sum_in(const Term* t, int n, wide low, wide high, int64_t& steps) {
  if (n == 0) return low < 0 && 0 < high;
  wide least = 0, most = 0;  // of the smaller ones
  for (int i = 1; i < n; ++i) { least += t[i].lo * t[i].stride; most += t[i].hi * t[i].stride; }
  // x * stride > low - most and x * stride < high - least
  const wide s = t[0].stride, above = low - most, below = high - least;
  const auto floor_div = [](wide a, wide b) { return a / b - (a % b < 0); };
  const wide first = floor_div(above, s) + 1 > t[0].lo ? floor_div(above, s) + 1 : t[0].lo;
  const wide last = -floor_div(-below, s) - 1 < t[0].hi ? -floor_div(-below, s) - 1 : t[0].hi;
  if (n == 1) return first <= last;
  for (wide x = first; x <= last; ++x) {
    if (--steps < 0) return true;
    if (some_sum_in(t + 1, n - 1, low - x * s, high - x * s, steps)) return true;
  }
  return false;
}
constexpr int64_t kSearchSteps = 1 << 16;

struct Terms {
  Term t[6];
  int n = 0;
  void add(wide stride, wide lo, wide hi) {
    if (stride == 0 || lo == hi) return;  // (lo == hi only for 0)
    int i = 0;
    while (i < n && t[i].stride > stride) ++i;
    if (i < n && t[i].stride == stride) { t[i].lo += lo; t[i].hi += hi; return; }
    for (int j = n++; j > i; --j) t[j] = t[j - 1];
    t[i] = {stride, lo, hi};
  }
};
inline bool empty(const Memory& m) { return !m.base || m.run <= 0 || m.count[0] <= 0 || m.count[1] <= 0 || m.count[2] <= 0; }
inline wide end_of(const Memory& m) {  // behind its last byte
  wide e = (wide)(uintptr_t)m.base + m.run;
  for (int d = 0; d < 3; ++d) e += (wide)(m.count[d] - 1) * m.stride[d];
  return e;
}
}  // namespace apart

// Whether a byte belongs to both (null or empty memory shares none).  Exact
// where strides are equal or nest, as those of one tensor's views do, whatever
// their ranges: columns of one projection are apart.  Takes nanoseconds where the
// ranges are apart; strides that would need a long search count as sharing.
inline bool share_bytes(const Memory& a, const Memory& b) {
  using namespace apart;
  if (empty(a) || empty(b)) return false;
  const wide at = (wide)(uintptr_t)b.base - (wide)(uintptr_t)a.base;
  if (end_of(a) <= (wide)(uintptr_t)b.base || end_of(b) <= (wide)(uintptr_t)a.base) return false;
  Terms t;
  for (int d = 0; d < 3; ++d) {
    t.add(b.stride[d], 0, b.count[d] - 1);
    t.add(a.stride[d], -(wide)(a.count[d] - 1), 0);
  }
  // a run of b starts less than a run of either before or behind one of a
  int64_t steps = kSearchSteps;
  return some_sum_in(t.t, t.n, -(wide)b.run - at, (wide)a.run - at, steps);
}

// Whether two runs of `a` share a byte.
inline bool shares_own_bytes(const Memory& a) {
  using namespace apart;
  if (empty(a)) return false;
  int64_t steps = kSearchSteps;
  for (int d = 0; d < 3; ++d) {  // two runs that differ in dimension d and in those behind it at will
    if (a.count[d] <= 1) continue;
    if (a.stride[d] == 0) return true;
    Terms t;
    for (int e = d + 1; e < 3; ++e) t.add(a.stride[e], -(wide)(a.count[e] - 1), a.count[e] - 1);
    // x * stride[d] for x >= 1, the others on either side: shifted by one stride to start at 0
    if (a.count[d] > 2) t.add(a.stride[d], 0, a.count[d] - 2);
    if (some_sum_in(t.t, t.n, -(wide)a.run - a.stride[d], (wide)a.run - a.stride[d], steps)) return true;
  }
  return false;
}

}  // namespace ennx
