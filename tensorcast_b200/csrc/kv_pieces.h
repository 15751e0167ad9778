// Where a range of tiles ends its pieces: a piece is what the range holds of one sequence.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define TCX_HOST_DEVICE __host__ __device__
#else
#define TCX_HOST_DEVICE
#endif

namespace tcx {

struct TileEnd {
  bool last, whole;  // of its piece; a piece that is its sequence whole
};

// Tile i of a range of `count` tiles that begins with tile `tile` of sequence `seq`,
// where tiles(s) is how many sequence s has.
template <typename Tiles>
TCX_HOST_DEVICE inline TileEnd tile_end(uint32_t seq, uint32_t tile, uint32_t count, uint32_t i, Tiles tiles) {
  uint32_t s = seq, t = tile + i, n = tiles(s);
  while (t >= n) {
    t -= n;
    n = tiles(++s);
  }
  const bool done = t + 1 == n;
  return {done || i + 1 == count, done && (s != seq || tile == 0)};
}

}  // namespace tcx
