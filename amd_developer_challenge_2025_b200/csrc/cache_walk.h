// How the tiles of a batch of cached sequences are shared out, for the kernels of mla_cache_sm100.cu and a host test.
//
// A sequence of n rows has ceil(n / 64) tiles; the tiles of all sequences lie one behind the other, and worker g of `workers`
// takes [share_begin(g), share_begin(g + 1)) of them, whatever sequences these belong to: shares differ by one tile at most,
// however ragged the batch is. A sequence that lies in the shares of several workers leaves a part with each of them.
#ifndef B200_CACHE_WALK_H_
#define B200_CACHE_WALK_H_

#ifdef __CUDACC__
#define CACHE_WALK_FN __host__ __device__ __forceinline__
#else
#define CACHE_WALK_FN inline
#endif

namespace cache_walk {

constexpr int kTileRows = 64;

CACHE_WALK_FN int tiles_of(int rows) { return (rows + kTileRows - 1) / kTileRows; }

// Workers that get tiles: as many as there are, but each with `least` tiles where the batch has that many.
CACHE_WALK_FN int workers_of(long long tiles, int most, int least) {
  const long long want = (tiles + least - 1) / least;
  return want < 1 ? 1 : want < most ? static_cast<int>(want) : most;
}

CACHE_WALK_FN long long share_begin(long long tiles, int workers, int g) { return tiles * g / workers; }

// The worker in whose share tile t lies (0 <= t < tiles).
CACHE_WALK_FN int worker_of(long long tiles, int workers, long long t) {
  return static_cast<int>(((t + 1) * workers - 1) / tiles);
}

// A worker's parts of split sequences: 0 for the one its share begins with, 1 for one that begins inside its share.
CACHE_WALK_FN int part_slot(long long share, long long first_tile_of_sequence) { return share >= first_tile_of_sequence ? 0 : 1; }

// Rows that one copy can bring: the largest power of two, at most a tile's, that divides the page, so that no copy crosses a
// page's end and every copy of a tile begins at a multiple of it.
CACHE_WALK_FN int copy_rows(int page_size) {
  int r = 1;
  while (r < kTileRows && page_size % (2 * r) == 0) r *= 2;
  return r;
}

}  // namespace cache_walk

#endif  // B200_CACHE_WALK_H_
