// How the tiles of a batch of cached sequences are shared out, for the kernels of mla_cache_sm100.cu and a host test.
//
// A sequence of n rows has ceil(n / tile) tiles, and costs `extra` tiles more to begin and end. On a line, every sequence that has
// rows takes its extra places and then one for each tile, and worker g of `workers` takes the places [share_begin(g), share_begin(g +
// 1)), whatever sequences these belong to: shares differ by one place at most, however ragged the batch is. A sequence whose tiles lie
// in the shares of several workers leaves a part with each of them; a border among the extra places splits nothing, and a sequence of
// few tiles goes whole to the worker that has its middle.
#ifndef B200_CACHE_WALK_H_
#define B200_CACHE_WALK_H_

#ifdef __CUDACC__
#define CACHE_WALK_FN __host__ __device__ __forceinline__
#else
#define CACHE_WALK_FN inline
#endif

namespace cache_walk {

CACHE_WALK_FN int tiles_of(int rows, int tile) { return (rows + tile - 1) / tile; }

// Places on the line of a sequence.
CACHE_WALK_FN int places_of(int rows, int tile, int extra) { return rows > 0 ? tiles_of(rows, tile) + extra : 0; }

// Workers that get a share: as many as there are, but each with `least` places where the batch has that many.
CACHE_WALK_FN int workers_of(long long places, int most, int least) {
  const long long want = (places + least - 1) / least;
  return want < 1 ? 1 : want < most ? static_cast<int>(want) : most;
}

CACHE_WALK_FN long long share_begin(long long places, int workers, int g) {
  // (a division in 64 bits takes the device several times as long)
  if (places < (1 << 20) && workers < (1 << 11)) return static_cast<unsigned>(places) * static_cast<unsigned>(g) / static_cast<unsigned>(workers);
  return places * g / workers;
}

// The worker in whose share place t lies (0 <= t < places).
CACHE_WALK_FN int worker_of(long long places, int workers, long long t) {
  return static_cast<int>(((t + 1) * workers - 1) / places);
}

constexpr int kWholeTiles = 4;  // 128 sequences of 60 rows, 32 heads: 20.6 us split evenly, 16.2 whole

// Places of a sequence whose holders have its first and its last part.
CACHE_WALK_FN long long first_place(long long begin, int tiles, int extra) { return begin + extra + (tiles <= kWholeTiles ? tiles / 2 : 0); }
CACHE_WALK_FN long long last_place(long long begin, int tiles, int extra) { return begin + extra + (tiles <= kWholeTiles ? tiles / 2 : tiles - 1); }

// The tiles [*first, *first + return value) of a sequence, whose places begin at `begin`, that the worker with the share [from, to) has.
CACHE_WALK_FN int tiles_in(long long begin, int tiles, int extra, long long from, long long to, int* first) {
  const long long t0 = begin + extra, t1 = t0 + tiles;
  if (tiles <= kWholeTiles) {
    const long long middle = first_place(begin, tiles, extra);
    *first = 0;
    return from <= middle && middle < to ? tiles : 0;
  }
  const long long a = from > t0 ? from : t0, b = to < t1 ? to : t1;
  *first = static_cast<int>(a - t0);
  return b > a ? static_cast<int>(b - a) : 0;
}

// Where a worker leaves its part of a split sequence: 0 where its share begins among the sequence's places, else 1.
CACHE_WALK_FN int part_slot(long long from, long long begin) { return from >= begin ? 0 : 1; }

// Rows that one copy can bring: the largest power of two that divides the tile and the page, so that no copy crosses a page's end
// and every copy of a tile begins at a multiple of it.
CACHE_WALK_FN int copy_rows(int page_size, int tile) {
  int r = 1;
  while (tile % (2 * r) == 0 && page_size % (2 * r) == 0) r *= 2;
  return r;
}

}  // namespace cache_walk

#endif  // B200_CACHE_WALK_H_
