// t5e_blocktiles.h -- what a results warp of the pair kernel does with the tiles
// behind one whose wait ran out: plain C++, so that it can be run without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define T5E_ANYWHERE __host__ __device__ __forceinline__
#else
#define T5E_ANYWHERE inline
#endif

namespace t5e {
namespace blockmm {

// write(row, col) for one lane's share of the tiles first, first + step, ... below
// `tiles`: of the warp's 32 rows from row0 of a tile of 256 rows by BN columns,
// the warp's 64 columns from col0 and, in a tile of 256, those 128 further on;
// a lane takes every 32nd column.
template <int BN, typename Write>
T5E_ANYWHERE void spoil_tiles(uint32_t first, uint32_t tiles, uint32_t step, uint32_t p_tiles, uint32_t row0, uint32_t col0,
                              uint32_t lane, uint32_t p_rows, uint32_t q_rows, Write write) {
  for (uint32_t tile = first; tile < tiles; tile += step) {
    const uint32_t p = tile % p_tiles * 256u + row0, q = tile / p_tiles * BN + col0 + lane;
    for (uint32_t i = 0; i < BN / 64 * 32u; ++i) {
      const uint32_t row = p + (i & 31u), col = q + (i >> 6) * 128u + (i >> 5 & 1u) * 32u;
      if (row < p_rows && col < q_rows) write(row, col);
    }
  }
}

}  // namespace blockmm
}  // namespace t5e
