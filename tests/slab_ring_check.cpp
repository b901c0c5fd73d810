// Walks a finishing warp's results through its slabs, for tiles of every kind: before a slab is written, each bulk store that was
// to read it has been waited for, whatever else left by bulk stores or without.
#include <cstdio>
#include <vector>

#include "slab_ring.h"

using namespace b200ta;

// The groups of a thread, in the order of their commits; a store reads its slab at the last moment that is allowed.
struct Groups {
  std::vector<std::vector<uint32_t>> pending;
  std::vector<uint32_t> open;
  int waited_for = -1;
  template <int kNewest>
  void wait_read() {
    while (int(pending.size()) > kNewest) pending.erase(pending.begin());
    waited_for = kNewest;
  }
  void commit() {
    pending.push_back(open);
    open.clear();
  }
  bool is_read(uint32_t slab) const {
    for (const auto& group : pending)
      for (uint32_t s : group)
        if (s == slab) return false;
    for (uint32_t s : open)
      if (s == slab) return false;
    return true;
  }
};

// `bulk`: for each result of a group of columns, whether it leaves by a bulk store; `tiles` tiles of `groups` such groups.
template <int kSlabs>
int check(const std::vector<bool>& bulk, int groups, int tiles) {
  SlabRing<kSlabs> ring;
  Groups queue;
  for (int n = 0; n < tiles * groups; ++n)
    for (size_t k = 0; k < bulk.size(); ++k) {
      bool free = false;
      uint32_t slab = 0;
      ring.pass(
          queue, [&](uint32_t s) { slab = s, free = s < kSlabs && queue.is_read(s); },
          [&](uint32_t s) {
            if (bulk[k]) queue.open.push_back(s);
          });
      if (!free) return std::printf("slab %u of %d is written before it is read: group %d, result %d\n", slab, kSlabs, n, int(k));
    }
  // no more waiting than the ring needs: as many groups may be pending as there are other slabs
  return queue.waited_for == kSlabs - 1 ? 0 : std::printf("waits for all but %d of %d slabs\n", queue.waited_for, kSlabs);
}

int main() {
  for (int groups : {1, 2, 3, 4, 8})
    for (int tiles : {1, 2, 3, 7}) {
      // results of a group of 32 columns: kept values in halves (dense: two; gated: of the value and the gate, four), then y;
      // or y alone, or dz of values and gates, or parts in 32 bits
      const std::vector<std::vector<bool>> two = {{true}, {false}, {true, true, true}, {true, true, false}, {true, false}};
      const std::vector<std::vector<bool>> three = {{true}, {false}, {true, true}, {true, true, true, true, true}, {true, true, true, true, false}, {true, true, false}};
      for (const auto& bulk : two)
        if (check<2>(bulk, groups, tiles) != 0) return 1;
      for (const auto& bulk : three)
        if (check<3>(bulk, groups, tiles) != 0) return 1;
    }
  std::puts("ok");
  return 0;
}
