// Whether two sets of evenly spaced rows have memory in common.  Integer code without CUDA or PyTorch, so that it compiles for a
// test by itself.
#pragma once
#include <algorithm>
#include <cstdint>

namespace b200ta_host {

// Rows of `bytes` bytes, `stride` bytes apart (not negative), the first one at `begin`.
struct RowSpan {
  int64_t begin, rows, bytes, stride;
};

// Whether a row of `b` has a byte of [begin, end).
inline bool overlaps_range(const RowSpan& b, int64_t begin, int64_t end) {
  if (b.begin >= end || b.begin + (b.rows - 1) * b.stride + b.bytes <= begin) return false;
  if (b.stride == 0 || b.begin + b.bytes > begin) return true;
  const int64_t first = (begin - b.begin - b.bytes) / b.stride + 1;  // the first row that ends behind `begin`
  return first < b.rows && b.begin + first * b.stride < end;
}

// A row of one and a row of the other.
inline bool overlaps(const RowSpan& a, const RowSpan& b) {
  if (a.rows <= 0 || b.rows <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
  if (a.rows > b.rows) return overlaps(b, a);
  if (a.begin >= b.begin + (b.rows - 1) * b.stride + b.bytes || b.begin >= a.begin + (a.rows - 1) * a.stride + a.bytes) return false;
  if (a.stride == b.stride && a.stride >= a.bytes) {
    // rows i of a and j of b overlap if -b.bytes < apart + t * stride < a.bytes with t = j - i
    const int64_t apart = b.begin - a.begin, stride = a.stride, low = -(a.rows - 1), high = b.rows - 1;
    auto floor_div = [](int64_t n, int64_t d) { return n / d - (n % d < 0); };
    const int64_t t0 = floor_div(-b.bytes - apart, stride) + 1, t1 = floor_div(a.bytes - apart - 1, stride);
    return std::max(t0, low) <= std::min(t1, high);
  }
  for (int64_t i = 0; i < a.rows; ++i)
    if (overlaps_range(b, a.begin + i * a.stride, a.begin + i * a.stride + a.bytes)) return true;
  return false;
}

}  // namespace b200ta_host
