// t5e_blocktiles.h -- the order in which a results warp of the pair kernel takes
// its tiles, apart from what it does with them: plain C++, so that what happens
// once a wait ran out can be run without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define T5E_ANYWHERE __host__ __device__ __forceinline__
#else
#define T5E_ANYWHERE inline
#endif

namespace t5e {
namespace blockmm {

// Tiles first, first + step, ... below `tiles`, the count-th of them by
// take(tile, count, ok) after wait(count).  Once a wait returned false no other
// is made, and every tile from there on is taken with ok = false: its results
// are still written (as NaN), so that none keeps what memory held before.
template <typename Wait, typename Take>
T5E_ANYWHERE bool take_tiles(uint32_t first, uint32_t tiles, uint32_t step, Wait wait, Take take) {
  bool ok = true;
  uint32_t count = 0;
  for (uint32_t tile = first; tile < tiles; tile += step, ++count) {
    ok = ok && wait(count);
    take(tile, count, ok);
  }
  return ok;
}

}  // namespace blockmm
}  // namespace t5e
