// How a place that is handed over again and again is told from its last time.  No CUDA in here: the order of events that
// follows is searched through on the CPU (tests/hand_over.cpp).
//
// A wait on an mbarrier names a phase by its parity alone: who looks when two phases have passed takes the one that runs
// for the one that was meant, and waits for a third.  One barrier is enough only where the side that arrives is kept from
// arriving twice before the other has looked.  Where it is not, but is never two pieces ahead, two barriers take turns: a
// barrier's next phase belongs to the piece after the next one, and cannot end before.
#pragma once
#include <cstdint>

#ifndef __CUDACC__
#define CSW_BOTH_SIDES
#else
#define CSW_BOTH_SIDES __host__ __device__ __forceinline__
#endif

namespace csw {

// Two barriers, 8 bytes apart, for the pieces 0, 1, 2, ... of a CTA.
struct Turns {
  uint32_t first;
  CSW_BOTH_SIDES uint32_t bar(uint32_t piece) const { return first + 8 * (piece % 2); }
  CSW_BOTH_SIDES static uint32_t parity(uint32_t piece) { return piece / 2 % 2; }
};

}  // namespace csw

#undef CSW_BOTH_SIDES
