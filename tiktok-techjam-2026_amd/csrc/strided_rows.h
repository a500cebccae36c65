// Whether strided rows share memory: host checks of what a call writes.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <utility>

namespace tjk {

// Rows of `bytes` bytes at base + sum of index * stride (bytes, none negative), one
// for each combination of the indexes below count.
struct StridedRows {
  static constexpr int kMost = 4;
  const void* base;
  int64_t bytes;
  int dims = 0;
  int64_t stride[kMost], count[kMost];
  StridedRows(const void* base, int64_t bytes) : base(base), bytes(bytes) {}
  StridedRows& by(int64_t step, int64_t n) {
    if (n > 1) stride[dims] = step, count[dims++] = n;
    return *this;
  }
};

namespace strided_rows {

typedef __int128 wide;  // (strides and counts are a caller's numbers: no sum of theirs overflows)

struct Step {
  int64_t stride, lo, hi;  // the multiples that may be taken
};

// Whether low < at + a multiple of each step < high is possible; steps of falling
// stride.  Of each only the multiples are tried that the smaller steps can bring back
// into the range: one or two, if rows nest.
inline bool lands(wide at, const Step* s, int n, wide low, wide high) {
  if (n == 0) return low < at && at < high;
  if (s->stride == 0) return lands(at, s + 1, n - 1, low, high);
  wide least = 0, most = 0;
  for (int i = 1; i < n; ++i) least += (wide)s[i].lo * s[i].stride, most += (wide)s[i].hi * s[i].stride;
  auto floor_div = [](wide a, int64_t b) { return a / b - (a % b < 0); };
  const wide from = std::max<wide>(floor_div(low - at - most, s->stride) + 1, s->lo);
  const wide to = std::min<wide>(-floor_div(at + least - high, s->stride) - 1, s->hi);
  for (wide d = from; d <= to; ++d)
    if (lands(at + d * s->stride, s + 1, n - 1, low, high)) return true;
  return false;
}

inline void sort(Step* s, int n) {
  std::sort(s, s + n, [](const Step& a, const Step& b) { return a.stride > b.stride; });
}

}  // namespace strided_rows

// Whether two of the rows share a byte.
inline bool rows_overlap(const StridedRows& r) {
  using namespace strided_rows;
  Step s[StridedRows::kMost];
  for (int i = 0; i < r.dims; ++i) s[i] = {r.stride[i], 1 - r.count[i], r.count[i] - 1};
  sort(s, r.dims);
  wide extent = r.bytes;  // of what the smaller steps reach
  int i = r.dims - 1;
  for (; i >= 0 && s[i].stride >= extent; --i) extent += (wide)s[i].hi * s[i].stride;
  if (i < 0) return false;  // each step is past all that the smaller ones reach
  for (i = 0; i < r.dims; ++i) {  // rows whose first differing index is the i-th
    s[i].lo = 1;
    if (lands(0, s + i, r.dims - i, -r.bytes, r.bytes)) return true;
  }
  return false;
}

// Whether a row of a and one of b share a byte.
inline bool rows_meet(const StridedRows& a, const StridedRows& b) {
  using namespace strided_rows;
  const wide at = (wide)(uintptr_t)a.base - (wide)(uintptr_t)b.base;
  wide a_extent = a.bytes, b_extent = b.bytes;
  for (int i = 0; i < a.dims; ++i) a_extent += (wide)(a.count[i] - 1) * a.stride[i];
  for (int i = 0; i < b.dims; ++i) b_extent += (wide)(b.count[i] - 1) * b.stride[i];
  if (at >= b_extent || -at >= a_extent) return false;
  Step s[2 * StridedRows::kMost];
  int n = 0;
  auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    for (int i = 0; i < n; ++i)
      if (s[i].stride == stride) {
        s[i].lo += lo, s[i].hi += hi;
        return;
      }
    s[n++] = {stride, lo, hi};
  };
  for (int i = 0; i < a.dims; ++i) add(a.stride[i], 0, a.count[i] - 1);
  for (int i = 0; i < b.dims; ++i) add(b.stride[i], 1 - b.count[i], 0);
  sort(s, n);
  return lands(at, s, n, -(wide)a.bytes, b.bytes);
}

}  // namespace tjk
