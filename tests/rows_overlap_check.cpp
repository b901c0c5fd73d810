// Compares the closed forms with marks on every byte, over a sweep of small sets of rows.
#include <cstdio>
#include <vector>

#include "rows_overlap.h"

using namespace b200ta_host;

static std::vector<int> marks(const RowSpan& a) {
  std::vector<int> m(400, 0);
  for (int64_t r = 0; r < a.rows; ++r)
    for (int64_t i = 0; i < a.bytes; ++i) ++m[a.begin + r * a.stride + i];
  return m;
}

int main() {
  std::vector<RowSpan> spans;
  for (int64_t rows : {0, 1, 2, 3, 5})
    for (int64_t bytes : {0, 1, 2, 3, 7, 12})
      for (int64_t stride : {0, 1, 3, 7, 8, 12, 20}) spans.push_back({0, rows, bytes, stride});
  for (RowSpan a : spans)
    for (RowSpan b : spans)
      for (int64_t at : {0, 1, 2, 5, 6, 7, 9, 13, 19, 20, 21, 37, 60, 90, 120}) {
        a.begin = 60, b.begin = at;
        const std::vector<int> x = marks(a), y = marks(b);
        bool common = false;
        for (size_t i = 0; i < x.size(); ++i) common |= x[i] > 0 && y[i] > 0;
        if (overlaps(a, b) != common || overlaps(b, a) != common)
          return std::printf("%d rows of %d, %d apart, and %d of %d, %d apart, at %d\n", int(a.rows), int(a.bytes), int(a.stride), int(b.rows),
                             int(b.bytes), int(b.stride), int(at - 60));
      }
  std::puts("ok");
  return 0;
}
