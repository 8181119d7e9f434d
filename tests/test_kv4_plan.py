"""The host arithmetic that plans blocks of positions over the 4-bit cache (shd_kv4.cuh), compiled by itself: costs of
very long caches must not pass 31 bits, and no tile costs more than the launch was planned for. No GPU needed."""
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <random>

#include "shd_kv4.cuh"
using namespace shd;

// Launches of M positions from pos0: every plan's sum and every tile's product with the heads in 31 bits.
static bool holds(const Kv4View& c, int M, int G, int pos0, int window, int tiles_most, bool every, int& launches) {
  const int step = kv4_launch_positions(c, M, G, pos0 + M - 1, tiles_most);
  if (step <= 0) return false;
  launches = 0;
  for (int m = 0; m < M; m += step, ++launches) {
    const int n = std::min(step, M - m), tiles = (int)(((int64_t)n * G + kKv4Tile - 1) / kKv4Tile);
    if (tiles > tiles_most) return false;
    int64_t sum = 0;
    for (int t = 0; t < tiles; ++t) {
      const int lo = pos0 + m + (int)((int64_t)t * kKv4Tile / G);
      const int hi = pos0 + m + std::min((int)(((int64_t)t * kKv4Tile + kKv4Tile - 1) / G), n - 1);
      if (!every && t > 0 && t + 1 < tiles) continue;
      const int64_t cost = kv4_tile_cost(c, lo, hi, window);
      sum += every ? cost : cost * tiles;  // the sampled tiles' costs bound the others' from both ends
      if (cost * c.heads > 0x7fffffff) return false;
    }
    if (!every) sum /= tiles > 1 ? 2 : 1;
    if (sum > 0x7fffffff) return false;
  }
  return true;
}

int main() {
  int launches = 0;
  Kv4View c{};
  // the last positions of caches of one head: 2^26 rows and more, with 2048 tiles, pass 2^31 in one launch
  for (int64_t cap : {int64_t(1) << 20, int64_t(1) << 26, int64_t(3) << 26, int64_t(1) << 28, int64_t(0x7ffffff0)}) {
    c.slots = 1, c.heads = 1, c.capacity = (int)cap, c.head_dim = 64, c.sinks = 0;
    const int M = 32768, pos0 = (int)(cap - M - 5);
    if (!holds(c, M, 8, pos0, 0, 2048, false, launches)) return printf("plan of %lld rows\n", (long long)cap), 1;
    printf("%lld %d\n", (long long)cap, launches);
  }
  // more heads than any memory holds rows for are refused
  c.capacity = 0x7ffffff0, c.heads = 64;
  if (kv4_launch_positions(c, 4, 1, 0x7fffffe0, 2048) != 0) return printf("64 heads\n"), 1;
  // ordinary ones go in one launch, up to the tiles that it takes
  c.capacity = 131072, c.heads = 8;
  if (kv4_launch_positions(c, 2048, 8, 131000, 2048) != 2048) return printf("one launch\n"), 1;
  if (kv4_launch_positions(c, 100000, 8, 131000, 2048) != 2048 * 128 / 8) return printf("tiles\n"), 1;
  // random settings, rings among them
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int i = 0; i < 20000; ++i) {
    c.heads = pick(1, 8);
    c.capacity = 16 * pick(1, 200);
    c.sinks = pick(0, std::min(40, c.capacity - 1));
    const int G = pick(1, 9), ring = c.capacity - c.sinks, M = pick(1, 200);
    const int pos0 = pick(0, 3 * c.capacity);
    int window = pick(0, 2 * c.capacity);
    if (pos0 + M > c.capacity) {
      if (M > ring) continue;
      window = pick(1, ring - M + 1);
    }
    if (!holds(c, M, G, pos0, window, pick(1, 64), true, launches)) return printf("setting %d\n", i), 1;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def planned(tmp_path_factory):
    from shardlm_b200 import build

    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cu").write_text(PROGRAM)
    subprocess.run([build._nvcc(), *build.ARCH_FLAGS, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-I", str(build.CSRC), "-I", str(ROOT / "include"),
                    "-o", str(at / "plan"), str(at / "plan.cu")], check=True, capture_output=True)
    return subprocess.run([str(at / "plan")], capture_output=True, text=True)


def test_plans_of_blocks_stay_in_range(planned):
    assert planned.returncode == 0, planned.stdout


def test_long_caches_take_more_launches(planned):
    launches = dict(map(int, line.split()) for line in planned.stdout.splitlines())
    assert launches[1 << 20] == 1  # 2048 tiles
    assert 1 < launches[1 << 26] <= 3 and launches[1 << 28] >= 4
