// The order in which a warp's results pass through its slabs of shared memory on their way out.  Integer code without CUDA
// calls, so that it also compiles for the host alone, where a test walks the slabs of every kind of tile.
//
// A slab is written, a bulk store reads it, and it may be written again only when that store has read it.  The hardware counts
// groups of stores and not slabs: before a slab is written, all groups but the newest kSlabs - 1 must have read theirs.  That
// means the slab's own last store only as long as every slab in turn has one group, so a result that leaves without a bulk store
// commits an empty one.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define B200TA_SLAB_RING __device__ __forceinline__
#else
#define B200TA_SLAB_RING inline
#endif

namespace b200ta {

template <int kSlabs>
struct SlabRing {
  uint32_t slot = 0;
  // One result: `write(slot)` fills the slab, `send(slot)` starts its store or stores it without a bulk store.  `groups` has
  // wait_read<n>() (all groups but the newest n have read their slabs) and commit().
  template <typename Groups, typename Write, typename Send>
  B200TA_SLAB_RING void pass(Groups&& groups, Write&& write, Send&& send) {
    groups.template wait_read<kSlabs - 1>();
    write(slot);
    send(slot);
    groups.commit();
    if (++slot == kSlabs) slot = 0;
  }
};

}  // namespace b200ta
