// The bound of a wait that may rightly last as long as the work of others: it counts polls in a row during which
// these did not move on, not polls.  Plain C++, so that it is tested without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define GDNX_WAIT_FN __host__ __device__ __forceinline__
#else
#define GDNX_WAIT_FN inline
#endif

namespace gdnx {
namespace pipe {

// Polls of a wait before it gives up.  A poll of a barrier to which nothing comes takes 4.0 us (measured, one warp or
// twelve): 17 s.
constexpr uint32_t kPolls = 1u << 22;

enum class Wait { kDone, kLeft, kRanOut };

// Polls done() until it is true, left() is true, or `polls` polls have passed since moved() last changed.
template <typename Done, typename Left, typename Moved>
GDNX_WAIT_FN Wait wait_while_moving(Done done, Left left, Moved moved, uint32_t polls) {
  uint32_t was = moved();
  for (uint32_t it = 0; it < polls; ++it) {
    if (done()) return Wait::kDone;
    if (left()) return Wait::kLeft;
    const uint32_t now = moved();
    if (now != was) {
      was = now;
      it = 0;
    }
  }
  return Wait::kRanOut;
}

}  // namespace pipe
}  // namespace gdnx
