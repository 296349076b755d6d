// The largest launch. Host code without HIP headers.
#pragma once

#include <cstdint>

namespace oxi {

// A dispatch counts the threads of a grid dimension in 32 bits. HIP refuses a
// launch of 2^32 of them or more, or runs it cut off and reports nothing (seen
// with 2^24 + 7 blocks of 256), and refuses 2^31 blocks or more.
inline int64_t most_blocks(int64_t threads) {
  const int64_t most = 0xffffffffll / threads;
  return most < ((int64_t)1 << 31) ? most : ((int64_t)1 << 31) - 1;
}
inline bool grid_fits(int64_t blocks, int64_t threads) {
  return blocks <= most_blocks(threads);
}

}  // namespace oxi
