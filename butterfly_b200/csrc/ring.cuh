// ring.cuh — slots of a shared-memory ring fed by asynchronous copies, and the log of which copies
// may still be in flight.  Host-callable too, so that the bookkeeping can be tested without a GPU.
#pragma once

#ifdef __CUDACC__
#define BNA_HD __host__ __device__ __forceinline__
#else
#define BNA_HD inline
#endif

namespace bna {

// WARPS consumer warps with SLOTS / WARPS slots each.  A barrier's parity tells a wait that is one use
// ahead nothing about the use before (copies complete out of order), so a slot stays with one
// warp.
template <int WARPS, int SLOTS>
struct Ring {
  static_assert(SLOTS % WARPS == 0, "a slot belongs to one warp");
  static constexpr int kUses = SLOTS / WARPS;  // uses of a warp until its first slot comes again
  BNA_HD static int slot(int use, int warp) { return use % kUses * WARPS + warp; }
  BNA_HD static unsigned parity(int use) { return (unsigned)(use / kUses) & 1u; }

  // The log: entry s is 1 + the last use whose copy went into slot s (0: none yet).  The copy before it
  // in the slot has landed, as the slot was free again.
  BNA_HD static void log(int* issued, int use, int warp) { issued[slot(use, warp)] = use + 1; }
  // wait(slot, parity) for the last copy into each slot; lane `lane` of `lanes` takes its share of the
  // slots.  Holds whichever copies were issued, in whatever order the lanes gave up.
  template <class Wait>
  BNA_HD static void settle(const int* issued, int lane, int lanes, Wait wait) {
    for (int s = lane; s < SLOTS; s += lanes)
      if (issued[s] > 0) wait(s, parity(issued[s] - 1));
  }
};

}  // namespace bna
