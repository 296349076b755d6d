// How the slices of a gradient list go over launches. Host code without HIP headers.
#pragma once

#include <cstdint>

#include "launch_limits.h"

namespace oxi {

// Of slices of size(0) .. size(count - 1) elements, cut into chunks of `chunk`, a block of `threads` each: calls
// add(slice, first element, elements, chunks) for each piece of a slice, in order or from the last slice's end
// on, and flush() behind the pieces of each launch: at most `most` of them, in a grid that a launch can have. A
// slice is one piece, unless its chunks alone pass that grid: then it is cut between chunks.
template <class Size, class Add, class Flush>
void walk_slices(Size size, int count, int64_t chunk, int threads, int most, bool back, Add add, Flush flush) {
  const int64_t room = most_blocks(threads);
  int64_t blocks = 0;
  int pieces = 0;
  auto end_launch = [&]() {
    if (pieces) flush();
    blocks = 0;
    pieces = 0;
  };
  for (int j = 0; j < count; ++j) {
    const int i = back ? count - 1 - j : j;
    const int64_t n = size(i), chunks = n / chunk + (n % chunk != 0), cuts = chunks / room + (chunks % room != 0);
    for (int64_t k = 0; k < cuts; ++k) {
      const int64_t first = (back ? cuts - 1 - k : k) * room;
      const int64_t nb = chunks - first < room ? chunks - first : room;
      if (pieces == most || nb > room - blocks) end_launch();
      const int64_t e0 = first * chunk;
      add(i, e0, n - e0 < nb * chunk ? n - e0 : nb * chunk, nb);
      blocks += nb;
      ++pieces;
    }
  }
  end_launch();
}

}  // namespace oxi
