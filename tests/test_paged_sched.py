"""The cutting of a paged_attention call, on the CPU: the header's plain functions are compiled with the
host compiler and run over random lengths (and lengths that are none)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = r"""
#include "paged_sched.hpp"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main(int argc, char **argv) {
  std::mt19937 rng(std::atoi(argv[1]));
  auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (uint32_t)(hi - lo + 1)); };
  for (int round = 0; round < 400; ++round) {
    const bool wild = round % 4 == 3;  // lengths that are none
    PagedSched c{};
    c.n_seqs = pick(1, 90);
    c.group = pick(1, 16);
    const bool decode = pick(0, 1);
    c.rows_over = decode ? 0 : pick(0, 1) * 16;
    c.rows_upto = decode ? 16 : 0x7fffffff;
    c.tile_rows = decode ? 16 : 128;
    c.align = decode ? 32 : 64;
    c.unit = decode ? 128 : 0;
    c.min_share = decode ? 2 : 512;
    c.target = pick(1, 96);
    c.alone = c.target / 2;
    c.rooms = decode ? c.target : 1 << 30;
    c.cut_cost = pick(0, 3) ? pick(0, 1300) : -1;
    c.window = pick(0, 2) ? 0 : pick(1, 500);
    c.max_len = pick(1, 1 << 14);
    std::vector<int> cu(c.n_seqs + 1), kv(c.n_seqs);
    for (int s = 0; s < c.n_seqs; ++s) {
      const int fresh = pick(0, 2) == 0 ? pick(0, 3) : pick(0, decode ? 5 : 300);
      cu[s + 1] = cu[s] + fresh;
      kv[s] = fresh + pick(0, 5000);
      if (pick(0, 9) == 0) kv[s] = pick(0, fresh);
    }
    c.n_tokens = cu[c.n_seqs] + pick(0, 5);
    if (wild)
      for (int s = 0; s < c.n_seqs; ++s) {
        cu[s] = (int)rng();
        kv[s] = (int)rng();
      }
    int64_t work = 0, tiles = 0, longest = 0;
    std::vector<PagedCost> cost(c.n_seqs);
    std::vector<int64_t> start(c.n_seqs + 1);
    for (int s = 0; s < c.n_seqs; ++s) {
      const PagedSeq q = sched_seq(c, cu[s], cu[s + 1], kv[s]);
      CHECK(0 <= q.q_begin && q.q_begin <= q.q_end && q.q_end <= c.n_tokens);
      CHECK(0 <= q.len && q.len <= c.max_len);
      CHECK(0 <= q.key_begin && q.key_begin <= q.key_end && q.key_end <= q.len && q.key_begin % c.align == 0);
      if (!wild)  // every key any row sees lies in the range
        for (int i = 0; i < q.q_end - q.q_begin; i += 7) {
          const int pos = q.pos0 + i;
          CHECK(pos == kv[s] - (cu[s + 1] - cu[s]) + i);
          const int hi = std::min(pos, q.len - 1), lo = c.window > 0 ? std::max(0, pos - c.window + 1) : 0;
          if (hi >= lo) CHECK(q.key_begin <= lo && hi < q.key_end);
        }
      cost[s] = sched_cost(c, q);
      const int64_t rows = (int64_t)(q.q_end - q.q_begin) * c.group;
      const bool in = rows > c.rows_over && rows <= c.rows_upto;
      CHECK((cost[s].tiles > 0) == in);
      if (in) {
        CHECK((int64_t)cost[s].tiles * c.tile_rows >= rows && (int64_t)(cost[s].tiles - 1) * c.tile_rows < rows);
        CHECK(cost[s].base >= 1 && cost[s].slope >= 0);
      }
      for (int t = 0; t < cost[s].tiles; ++t) CHECK(sched_before(cost[s], t + 1) - sched_before(cost[s], t) == cost[s].base + cost[s].slope * t);
      start[s] = work;
      work += sched_before(cost[s], cost[s].tiles);
      tiles += cost[s].tiles;
      if (cost[s].tiles) longest = std::max(longest, cost[s].base + cost[s].slope * (cost[s].tiles - 1));
    }
    start[c.n_seqs] = work;
    const int64_t share = sched_share(c, work);
    CHECK(share >= 1 && share * c.target >= work);
    const bool whole = sched_whole(c, tiles, work, longest);
    if (c.cut_cost < 0) CHECK(whole);
    else CHECK(!whole || tiles <= c.rooms);
    if (wild) continue;
    const int64_t bound = sched_tiles_bound(c, 0);
    CHECK(tiles <= bound);
    if (!whole) CHECK((work + share - 1) / share <= c.target);
    // a share begins at most one tile that it does not end: its parts have distinct slots
    if (!whole) {
      std::vector<int> used(sched_slots_bound(c), 0);
      for (int s = 0; s < c.n_seqs; ++s)
        for (int t = 0; t < cost[s].tiles; ++t) {
          const int64_t a = start[s] + sched_before(cost[s], t), b = a + cost[s].base + cost[s].slope * t;
          const int64_t first = a / share, last = (b - 1) / share;
          CHECK(last < c.target);
          if (first == last) continue;
          for (int64_t w = first; w <= last; ++w) {
            const int64_t from = std::max(a, w * share) - a;
            const int64_t slot = 2 * w + (from == 0 ? 1 : 0);
            CHECK(slot == 2 * w + (w == first ? 1 : 0) || w * share == a);
            CHECK(slot < (int64_t)used.size() && !used[slot]++);
          }
        }
    }
  }
  std::printf("ok\n");
  return 0;
}
"""


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_shares_cover_the_work_and_slots_do_not_collide(tmp_path, seed):
    src, exe = tmp_path / "s.cpp", tmp_path / "s"
    src.write_text(SRC)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                           os.path.join(HERE, "..", "argus-engine_amd", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe), str(seed)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]
