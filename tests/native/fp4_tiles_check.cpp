// Walks the tiles of the many-row FP4 product as its CTA pairs do, one step past the last tile included (built with
// -fsanitize=undefined): every tile exactly once, whatever the number of row pairs, columns and CTA pairs.
#include <cstdio>
#include <vector>

#include "../../wan-dit-lab_b200/csrc/fp4_tiles.h"

int main() {
  for (int m_pairs = 1; m_pairs <= 33; ++m_pairs)
    for (int n_tiles = 1; n_tiles <= 9; ++n_tiles) {
      const int tiles = m_pairs * n_tiles;
      for (int pairs : {1, 3, 74}) {
        std::vector<int> seen(tiles, 0);
        for (int pair = 0; pair < pairs && pair < tiles; ++pair) {
          int t = pair;
          for (; t < tiles; t += pairs) {
            const wdl::fp4::Tile tile = wdl::fp4::tile_of(t, m_pairs, n_tiles);
            if (tile.m_pair < 0 || tile.m_pair >= m_pairs || tile.n_tile < 0 || tile.n_tile >= n_tiles) return 1;
            ++seen[tile.n_tile * m_pairs + tile.m_pair];
          }
          volatile int past = wdl::fp4::tile_of(t, m_pairs, n_tiles).m_pair;
          (void)past;
        }
        for (int count : seen)
          if (count != 1) return 2;
      }
    }
  std::puts("ok");
  return 0;
}
