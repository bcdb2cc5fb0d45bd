// Argument checks of the entry points that need no CUDA header, so that they can
// be compiled and tested on their own.
#pragma once
#include <cstdint>

namespace flock {

// Positions pos .. pos + n - 1 lie inside a cache of `capacity` keys.  No sum of
// the caller's numbers: pos + n may pass 2^63.
inline bool range_inside(int64_t pos, int64_t n, int64_t capacity) {
  return pos >= 0 && n >= 0 && n <= capacity && pos <= capacity - n;
}

}  // namespace flock
