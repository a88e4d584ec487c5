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
// walk <most> <least> <rows of sequence 0> <rows of sequence 1> ...: per worker "worker begin end", then per part of a split sequence,
// as the attention writes them "w sequence worker slot first count", as the join looks them up "j sequence worker slot"
int main(int argc, char** argv) {
  const int most = atoi(argv[1]), least = atoi(argv[2]);
  std::vector<long long> first{0};
  for (int i = 3; i < argc; ++i) first.push_back(first.back() + tiles_of(atoi(argv[i])));
  const long long tiles = first.back();
  const int workers = workers_of(tiles, most, least);
  for (int g = 0; g < workers; ++g) {
    long long t = share_begin(tiles, workers, g);
    const long long end = share_begin(tiles, workers, g + 1);
    printf("%d %lld %lld\\n", g, t, end);
    for (int segment = 0; t < end; ++segment) {
      int b = 0;
      while (first[b + 1] <= t) ++b;
      const long long to = end < first[b + 1] ? end : first[b + 1];
      if (t != first[b] || to != first[b + 1]) printf("w %d %d %d %lld %lld\\n", b, g, segment == 0 ? 0 : 1, t - first[b], to - t);
      t = to;
    }
  }
  for (int b = 0; b + 3 < argc; ++b) {
    if (first[b] == first[b + 1]) continue;
    const int g0 = worker_of(tiles, workers, first[b]), g1 = worker_of(tiles, workers, first[b + 1] - 1);
    for (int g = g0; g1 > g0 && g <= g1; ++g) printf("j %d %d %d\\n", b, g, part_slot(share_begin(tiles, workers, g), first[b]));
  }
  for (int p = 1; p <= 300; ++p) printf("r %d %d\\n", p, copy_rows(p));
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


@pytest.mark.parametrize("most,least", [(1, 1), (2, 1), (74, 1), (148, 1), (148, 3), (512, 2)])
def test_shares_and_parts(walk, most, least):
    rng = random.Random(most + least)
    for rows in ([1], [64], [65], [0, 0], [0, 5, 0], [9000], [1] * 200, [rng.randint(0, 900) for _ in range(60)],
                 [rng.choice([0, 1, 64, 65, 20000]) for _ in range(30)]):
        lines = walk(most, least, *rows)
        shares = [tuple(map(int, f)) for f in lines if f[0].isdigit()]
        tiles = sum(-(-n // 64) for n in rows)
        assert 1 <= len(shares) <= most and shares[0][1] == 0 and shares[-1][2] == tiles
        assert all(a[2] == b[1] for a, b in zip(shares, shares[1:]))
        sizes = [e - b for _, b, e in shares]
        assert max(sizes) - min(sizes) <= 1
        assert len(shares) == 1 or tiles > (len(shares) - 1) * least
        written = [tuple(map(int, f[1:])) for f in lines if f[0] == "w"]
        assert [w[:3] for w in written] == sorted(w[:3] for w in written)
        assert [w[:3] for w in written] == [tuple(map(int, f[1:])) for f in lines if f[0] == "j"]
        assert len({w[1:3] for w in written}) == len(written)  # no two parts in one place
        for b in {w[0] for w in written}:
            at = 0
            for w in (w for w in written if w[0] == b):
                assert w[3] == at and w[4] > 0
                at += w[4]
            assert at == -(-rows[b] // 64)


def test_copies_stay_inside_their_page_and_tile(walk):
    lines = walk(1, 1, 1)
    assert ["far"] not in lines
    for _, page, rows in (f for f in lines if f[0] == "r"):
        page, rows = int(page), int(rows)
        assert page % rows == 0 and 64 % rows == 0 and (rows == 64 or page % (2 * rows) != 0)
