// How the two warps that share the rows of a tile exchange a value a row, inside a
// kernel whose waits are bounded.
//
// They meet at a barrier of the two, which has no limit of its own: both have to
// call it equally often, whatever their waits return.  One warp's wait can run out
// just before its partner sees the same phase complete, and a partner that finds a
// phase complete does not learn that anybody gave up.  So a warp whose wait ran out
// still meets its partner once, leaving a mark in place of its value, and both leave
// their loops after that one meeting.
//
// Nothing here needs the GPU: tests/test_pair_exchange_cpu.py compiles this file for
// the host and runs every order of waits that run out.
#pragma once

#include <math.h>

namespace theria {
namespace tc {

// A lane's value x (never NaN) goes to *mine, its partner's is read from *theirs into
// `other`.  `landed` (the same for a whole warp): this warp's wait returned in time.
// `meet` is the barrier of the two warps.  Returns whether both warps' waits did.
// Calls alternate between two places in memory, so that a value is read before the
// partner writes there again.
template <typename Meet>
__device__ __forceinline__ bool pair_exchange(float* mine, const float* theirs, bool landed,
                                              float x, float& other, Meet meet) {
  *mine = landed ? x : NAN;
  meet();
  other = *theirs;
  return landed && other == other;
}

}  // namespace tc
}  // namespace theria
