// The order in which the many-row FP4 product takes its output tiles (plain C++: the host's tests walk it too).
#pragma once

#ifdef __CUDACC__
#define WDL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define WDL_HOST_DEVICE inline
#endif

namespace wdl {
namespace fp4 {

// Tile t: row pairs fastest within groups of 8 of them, so that the tiles under way at one time share rows of a as well
// as of w in L2 however many rows there are. A t past the last tile, which a producer asks for after its last step, names
// no tile, but is computed without a division by zero (row pairs a multiple of 8).
struct Tile {
  int m_pair, n_tile;
};
WDL_HOST_DEVICE Tile tile_of(int t, int m_pairs, int n_tiles) {
  const int group = t / (8 * n_tiles), left = m_pairs - group * 8, rows = left < 1 ? 1 : left < 8 ? left : 8;
  const int r = t - group * 8 * n_tiles;
  return {group * 8 + r % rows, r / rows};
}

}  // namespace fp4
}  // namespace wdl
