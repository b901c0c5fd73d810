// Walks the windows of rows of numbered elements: each lies behind the last one, and together they are the row, also where elements'
// places pass 32 bits.
#include <cstdio>
#include <initializer_list>

#include "dropout_windows.h"

using namespace b200ta;

int main() {
  const int64_t two31 = int64_t(1) << 31;
  for (int64_t inner : {int64_t(16), int64_t(17), int64_t(2039), int64_t(2040), int64_t(2041), int64_t(4099), two31 - 1, two31 + 8, two31 + 4099, 2 * two31 + 7,
                        3 * two31 - 1}) {
    const int64_t windows = dropout_windows(inner);
    for (int64_t outer : {0, 1, 2}) {
      if ((outer + 1) * windows >= two31) break;  // (as many blocks as a launch may have)
      int64_t next = 0;
      for (int64_t w = 0; w < windows; ++w) {
        const DropoutWindow at = dropout_window(uint32_t(outer * windows + w), uint32_t(windows), inner);
        if (at.outer != outer || at.first != next || at.width < 1 || at.width > kDropoutWindow || at.first + at.width > inner)
          return std::printf("window %lld of row %lld of %lld elements: from %lld, %d\n", (long long)w, (long long)outer, (long long)inner, (long long)at.first,
                             at.width);
        next += at.width;
      }
      if (next != inner) return std::printf("%lld of %lld elements\n", (long long)next, (long long)inner);
    }
  }
  std::puts("ok");
  return 0;
}
