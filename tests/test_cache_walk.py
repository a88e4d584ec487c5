"""How the attention over a paged cache shares out its tiles, from the header that the kernels include: every tile has one
worker, shares differ by a tile at most, and the part of a sequence that a worker leaves is found again by the join."""
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd_developer_challenge_2025_b200", "csrc")
PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "cache_walk.h"
using namespace cache_walk;
// walk <most> <least> <tile> <extra> <rows of sequence 0> <rows of sequence 1> ...: per worker "worker places", per segment "s sequence worker
// first count", per part of a split sequence "w sequence worker slot first count" as the attention writes it, "j sequence worker slot" as
// the join looks it up
int main(int argc, char** argv) {
  const int most = atoi(argv[1]), least = atoi(argv[2]), tile = atoi(argv[3]), extra = atoi(argv[4]), batch = argc - 5;
  std::vector<int> rows;
  std::vector<long long> begins{0};
  for (int b = 0; b < batch; ++b) {
    rows.push_back(atoi(argv[5 + b]));
    begins.push_back(begins.back() + places_of(rows[b], tile, extra));
  }
  const long long places = begins.back();
  const int workers = workers_of(places, most, least);
  for (int g = 0; g < workers; ++g) {
    const long long from = share_begin(places, workers, g), to = share_begin(places, workers, g + 1);
    printf("%d %lld\\n", g, to - from);
    for (int b = 0; b < batch; ++b) {
      int first;
      const int count = rows[b] > 0 ? tiles_in(begins[b], tiles_of(rows[b], tile), extra, from, to, &first) : 0;
      if (count == 0) continue;
      printf("s %d %d %d %d\\n", b, g, first, count);
      if (count != tiles_of(rows[b], tile)) printf("w %d %d %d %d %d\\n", b, g, part_slot(from, begins[b]), first, count);
    }
  }
  for (int b = 0; b < batch; ++b) {
    if (begins[b] == begins[b + 1]) continue;
    const int tiles = tiles_of(rows[b], tile);
    const int g0 = worker_of(places, workers, first_place(begins[b], tiles, extra)), g1 = worker_of(places, workers, last_place(begins[b], tiles, extra));
    for (int g = g0; g1 > g0 && g <= g1; ++g) printf("j %d %d %d\\n", b, g, g == g0 ? part_slot(share_begin(places, workers, g), begins[b]) : 0);
  }
  for (int p = 1; p <= 300; ++p) printf("r %d %d\\n", p, copy_rows(p, tile));
  // far beyond 32 bits
  for (int g = 0; g < 148; ++g) {
    const long long many = (1ll << 24) * 65535;
    if (worker_of(many, 148, share_begin(many, 148, g)) != g || worker_of(many, 148, share_begin(many, 148, g + 1) - 1) != g) printf("far\\n");
  }
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(PROGRAM)
    subprocess.check_call([cxx, "-std=c++17", f"-I{CSRC}", str(d / "walk.cpp"), "-o", str(d / "walk")])
    return lambda *args: [line.split() for line in subprocess.check_output([str(d / "walk"), *map(str, args)], text=True).splitlines()]


@pytest.mark.parametrize("tile,extra", [(64, 0), (64, 2), (48, 1), (48, 0), (64, 5)])
@pytest.mark.parametrize("most,least", [(1, 1), (2, 1), (74, 1), (148, 1), (148, 3), (512, 2)])
def test_shares_and_parts(walk, most, least, tile, extra):
    rng = random.Random(most + least + extra)
    for rows in ([1], [64], [65], [0, 0], [0, 5, 0], [9000], [1] * 200, [rng.randint(0, 900) for _ in range(60)],
                 [rng.choice([0, 1, 64, 65, 20000]) for _ in range(30)], [60] * 128, [256, 257, 192, 193, 300] * 20):
        lines = walk(most, least, tile, extra, *rows)
        sizes = [int(f[1]) for f in lines if f[0].isdigit()]
        tiles = [-(-n // tile) for n in rows]
        places = sum(n + extra for n in tiles if n)
        assert 1 <= len(sizes) <= most and sum(sizes) == places
        assert max(sizes) - min(sizes) <= 1
        assert len(sizes) == 1 or places > (len(sizes) - 1) * least
        segments = [tuple(map(int, f[1:])) for f in lines if f[0] == "s"]
        for b, n in enumerate(tiles):  # every tile once, in the order of the workers
            at = 0
            for s in (s for s in segments if s[0] == b):
                assert s[2] == at and s[3] > 0
                at += s[3]
            assert at == n
            assert n > 4 or sum(s[0] == b for s in segments) <= 1
        written = [tuple(map(int, f[1:])) for f in lines if f[0] == "w"]
        assert [w[:3] for w in sorted(written)] == [tuple(map(int, f[1:])) for f in lines if f[0] == "j"]
        assert len({w[1:3] for w in written}) == len(written)  # no two parts in one place


@pytest.mark.parametrize("tile", [48, 64])
def test_copies_stay_inside_their_page_and_tile(walk, tile):
    lines = walk(1, 1, tile, 0, 1)
    assert ["far"] not in lines
    for _, page, rows in (f for f in lines if f[0] == "r"):
        page, rows = int(page), int(rows)
        assert page % rows == 0 and tile % rows == 0 and (tile % (2 * rows) != 0 or page % (2 * rows) != 0)
