// The host's questions about an index of adapters: the number that divides a row's by the rows of an entry, and the adapters of a tile.
#include <cstdio>

#include "adapters.cuh"

using namespace b200ta;

int main() {
  const int64_t top = (int64_t(1) << 31) - 1;
  for (int64_t d : {int64_t(1), int64_t(2), int64_t(3), int64_t(7), int64_t(23), int64_t(127), int64_t(128), int64_t(129), int64_t(36864), int64_t(147456),
                    (int64_t(1) << 30) + 1, top, top + 1, top * 4}) {
    const AdapterIndex x = adapter_index(&top, 8, d, 3);
    for (int64_t k : {int64_t(0), int64_t(1), int64_t(2), top / d / 2, top / d})
      for (int64_t e = -1; e <= 1; ++e) {
        const int64_t n = k * d + e;
        if (n < 0 || n > top) continue;
        if (int64_t(uint64_t(n) * x.factor >> x.shift) != n / d) return std::printf("row %lld of %lld to an entry\n", (long long)n, (long long)d);
      }
  }
  struct {
    bool index;
    int64_t rows_per_index, rows;
    int count, tile, want;
  } const tiles[] = {
      {false, 0, 1000, 1, 128, 1},      {false, 0, 1000, 1, 256, 1},  {true, 1, 4000, 100, 128, 100}, {true, 1, 4000, 1000, 128, 128},
      {true, 1, 4000, 1000, 256, 256},  {true, 1, 20, 64, 128, 20},   {true, 1, 20, 64, 256, 20},     {true, 16, 4000, 1000, 128, 8},
      {true, 16, 4000, 1000, 256, 16},  {true, 100, 4000, 9, 128, 2}, {true, 100, 4000, 9, 256, 3},   {true, 200, 4000, 9, 128, 1},
      {true, 200, 4000, 9, 256, 2},     {true, 200, 200, 9, 256, 1},  {true, 36864, 300000, 9, 256, 1},
  };
  for (const auto& t : tiles) {
    const AdapterIndex x = adapter_index(t.index ? &top : nullptr, 4, t.rows_per_index, t.count);
    if (adapters_of_tile(x, t.rows, t.tile) != t.want)
      return std::printf("%lld rows, %lld to an entry, %d adapters: tiles of %d have %lld\n", (long long)t.rows, (long long)t.rows_per_index, t.count, t.tile,
                         (long long)adapters_of_tile(x, t.rows, t.tile));
  }
  std::puts("ok");
  return 0;
}
