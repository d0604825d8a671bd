"""CPU proof of the order in which the expanded attention takes its query tiles.

Compiles ferret_amd/csrc/expanded_plan.hpp with g++ and walks the kernel's search
(expanded_attention.hip) for every start slot of many ragged batches: every tile
of every sequence is taken once, by falling numbers of steps over the ranks.
"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ferret_amd", "csrc")

WALKER = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>
#include "expanded_plan.hpp"
using namespace ferret;

static long long bad = 0;
#define CHECK(c) do { if (!(c) && bad++ < 20) std::printf("line %d: %s\n", __LINE__, #c); } while (0)

static int steps_of(const TileSeq& s, int tile) {
  const int end = std::min(kTileTokens * (tile + 1), s.n), sees = s.causal ? std::max(s.len - s.n + end, 0) : s.len;
  return (std::min(sees, s.len) + kTileKeys - 1) / kTileKeys;
}

int main() {
  std::srand(5);
  auto pick = [](int lo, int hi) { return lo + std::rand() % (hi - lo + 1); };
  for (int k = 0; k < 1500; ++k) {
    const int B = pick(1, kOrderedBatch), causal = pick(0, 3) != 0;
    std::vector<TileSeq> seqs;
    int S = 1, all = 0;
    for (int b = 0; b < B; ++b) {
      const int n = pick(0, 3) ? pick(0, 900) : pick(0, 2);
      seqs.push_back(TileSeq{n, std::max(0, n + pick(-200, k % 7 ? 2000 : 40000)), causal});
      S += seqs.back().len;
      all += seqs.back().tiles();
      for (int t = 0; t < 70; ++t) {
        int count = 0;
        for (int j = 0; j < seqs.back().tiles(); ++j) count += steps_of(seqs.back(), j) >= t;
        CHECK(seqs.back().at_least(t) == count);
      }
    }
    std::set<std::pair<int, int>> taken;
    std::map<int, int> by_rank;
    for (int slot = 0; slot < all; ++slot) {
      const int rank = slot;
      int base = 0, stride = (S + kTileKeys - 1) / kTileKeys / 64 + 1;
      for (;;) {
        int top = -1;
        for (int lane = 0; lane < 64; ++lane) {
          int count = 0;
          for (const auto& s : seqs) count += s.at_least(base + lane * stride);
          if (count > rank) top = lane;
        }
        CHECK(top >= 0);
        base += top * stride;
        if (stride == 1) break;
        stride = (stride + 63) / 64;
      }
      int before = 0, b = -1, tile = 0;
      for (const auto& s : seqs) before += s.at_least(base + 1);
      int among = rank - before;
      for (int i = 0; i < B && b < 0; ++i) {
        const int from = seqs[i].first_of(base), count = seqs[i].first_of(base + 1) - from;
        if (among < count) { b = i; tile = from + among; }
        among -= count;
      }
      CHECK(b >= 0 && tile >= 0 && tile < seqs[b].tiles() && taken.insert({b, tile}).second);
      if (b >= 0) CHECK(steps_of(seqs[b], tile) == base);
      by_rank[rank] = base;
    }
    CHECK((int)taken.size() == all && (int)by_rank.size() == all);
    for (int r = 1; r < all; ++r) CHECK(by_rank[r] <= by_rank[r - 1]);
  }
  for (int all = 1; all < 700; all += 13)  // the ranks of paired work-groups: each once
    for (int first : {0, 1, 2, 16, 32, 256}) {
      std::set<int> ranks;
      for (int slot = 0; slot < all; ++slot) ranks.insert(paired_rank(slot, all, first));
      CHECK((int)ranks.size() == all && *ranks.begin() == 0 && *ranks.rbegin() == all - 1);
    }
  std::printf("%lld violations\n", bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_every_tile_once_longest_first(tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(WALKER)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}",
                    str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.endswith("0 violations\n")
