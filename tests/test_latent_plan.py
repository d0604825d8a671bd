"""CPU proof of how the latent attention deals its work and finds its rows.

Compiles ferret_amd/csrc/latent_plan.hpp with g++ together with a walker that
follows the kernel's loop (latent_attention.hip) for every work-group of many
ragged batches, index tensors with values outside their tensors among them:
every (sequence, row tile, step) is taken exactly once, pieces of one tile have
slots of their own inside the workspace, the record of a tile leads to its
pieces in order, query rows stay inside [0, T * H), and no page entry leads to a
row outside the cache.
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
#include <tuple>
#include <vector>
#include <climits>
#include "latent_plan.hpp"
using namespace ferret;

static long long bad = 0, walked = 0, whole = 0, cut = 0;
#define CHECK(c) do { if (!(c) && bad++ < 20) std::printf("line %d: %s\n", __LINE__, #c); } while (0)

static void walk(const std::vector<int>& cu, const std::vector<int>& lens, int T, int H, int mr, int side, int most,
                 int min_steps) {
  const int B = (int)lens.size(), units = kLatentUnits / side;
  auto seq = [&](int b) { return latent_seq(cu[b], cu[b + 1], lens[b], T, H, mr, side, most); };
  int total = 0, groups = 0;
  const int threads = mr == 16 ? 256 : 512;
  for (int b = 0; b < B; ++b) {
    const LatentSeq s = seq(b);
    CHECK(s.q0 >= 0 && s.n >= 0 && s.q0 + s.n <= T && s.len >= 0 && s.len <= most && s.steps >= 1);
    CHECK((long long)s.groups * mr * side >= s.rows && (s.groups == 0 || (s.groups - 1) * mr * side < s.rows));
    total += s.work(0);
    groups += s.groups;
  }
  int chunk = latent_chunk(total, units, min_steps), extra = kLatentExtra;
  bool fits = B <= threads;
  for (int b = 0; b < B; ++b) fits = fits && latent_fits(seq(b), chunk);
  if (fits) extra = 0;
  total += extra * groups;
  if (extra != 0) chunk = latent_chunk(total, units, min_steps);
  (fits ? whole : cut) += 1;
  long long expected = 0;
  std::set<std::tuple<int, int, int>> done;
  std::map<std::pair<int, int>, std::vector<std::pair<int, int>>> pieces;  // tile -> (first step, slot)
  std::map<std::pair<int, int>, LatentRecord> records;
  std::set<int> slots;
  std::set<std::pair<int, int>> places;
  for (int block = 0; block < kLatentUnits; ++block) {
    const LatentPlace at = latent_place(block, side);
    CHECK(at.unit >= 0 && at.unit < units && at.lane >= 0 && at.lane < side && places.insert({at.unit, at.lane}).second);
    CHECK(at.unit % 8 == block % 8);  // one XCD
    const int start = (int)((long long)at.unit * chunk < total ? (long long)at.unit * chunk : total);
    if (start >= total) continue;
    const int end = plan_min(start + chunk, total);
    int b = 0, seq_at = 0, cur = start;
    while (seq_at + seq(b).work(extra) <= start) seq_at += seq(b++).work(extra);
    while (cur < end) {
      LatentSeq s = seq(b);
      while (cur >= seq_at + s.work(extra) && b + 1 < B) {
        seq_at += s.work(extra);
        s = seq(++b);
      }
      const int line = s.steps + extra, group = s.groups > 1 ? (cur - seq_at) / line : 0;
      const int s0 = cur - seq_at - group * line, s1 = plan_min(line, s0 + end - cur);
      const int tile = group * side + at.lane;
      CHECK(group >= 0 && group < s.groups && s0 >= 0 && s1 > s0);
      const int row0 = tile * mr, row_last = plan_min(row0 + mr, s.rows) - 1;
      if (row_last < row0 || s0 >= s.steps) {
        cur += s1 - s0;
        continue;
      }
      CHECK(row_last >= row0 && (long long)s.q0 * H + row_last < (long long)T * H);
      for (int t = s0; t < plan_min(s1, s.steps); ++t) CHECK(done.insert({b, tile, t}).second);
      if (!(s0 == 0 && s1 >= s.steps)) {
        const int slot = latent_slot(at.unit, at.lane, side, cur, chunk);
        CHECK(slot >= 0 && slot < 2 * kLatentUnits && slots.insert(slot).second);
        pieces[{b, tile}].push_back({s0, slot});
      }
      if (s0 == 0) records[{b, tile}] = latent_record(at.unit, at.lane, side, cur, s.steps, chunk);
      cur += s1 - s0;
    }
  }
  for (int b = 0; b < B; ++b)
    for (int tile = 0; tile * mr < seq(b).rows; ++tile) {
      expected += seq(b).steps;
      CHECK(records.count({b, tile}) == 1);
      const LatentRecord r = records[{b, tile}];
      auto& p = pieces[{b, tile}];
      std::sort(p.begin(), p.end());
      CHECK(latent_record_joins(r, side) == (p.size() > 0));
      if (p.empty()) {
        CHECK(r.pieces == 1);
        continue;
      }
      CHECK((int)p.size() == r.pieces);  // units ascend, so do the steps
      for (int j = 0; j < r.pieces && j < (int)p.size(); ++j)
        CHECK(p[j].second == latent_record_slot(r, side, j) && (j == 0) == (p[j].first == 0));
    }
  CHECK((long long)done.size() == expected);
  ++walked;
}

int main() {
  std::srand(7);
  auto pick = [](int lo, int hi) { return lo + std::rand() % (hi - lo + 1); };
  for (int k = 0; k < 1500; ++k) {
    const int B = k % 3 == 0 ? pick(1, 300) : pick(1, 20), H = pick(0, 2) ? pick(1, 40) : 128, mr = 16 << pick(0, 2);
    const int page = 16 * pick(1, 5), max_pages = pick(1, 60), most = page * max_pages;
    std::vector<int> cu{0}, lens;
    for (int b = 0; b < B; ++b) {
      const int n = pick(0, 3) ? pick(0, 2) : pick(0, 30);
      cu.push_back(cu.back() + n);
      lens.push_back(pick(0, 5) ? pick(0, most) : pick(-3, 3) * (INT_MAX / 4));
    }
    const int T = cu.back() + pick(0, 3) > 0 ? cu.back() + pick(1, 3) : 1;
    if (k % 10 == 9) for (auto& c : cu) if (!pick(0, 4)) c = pick(-5, T + 40) * (pick(0, 1) ? 1 : INT_MAX / (T + 60));
    const int side = 1 << pick(0, 3);
    if (k % 10 != 9) walk(cu, lens, T, H, mr, side, most, pick(1, 9));
    else for (int b = 0; b < B; ++b) {  // not ascending: rows stay inside all the same
      const LatentSeq s = latent_seq(cu[b], cu[b + 1], lens[b], T, H, mr, side, most);
      CHECK(s.q0 >= 0 && s.n >= 0 && s.q0 + s.n <= T && s.len >= 0 && s.len <= most);
    }
  }
  for (int pages : {1, 3, 1 << 20})
    for (int id : {INT_MIN, -1, 0, pages - 1, pages, pages + 1, INT_MAX}) {
      const long long r = page_row(id, pages, 64, 63);
      CHECK(r == (id >= 0 && id < pages ? (long long)id * 64 + 63 : -1));
    }
  for (int side : {1, 2, 4, 8})
    for (int v : {INT_MIN, -1, 0, 1, 254, 255, 256, 510, 511, 512, INT_MAX})
      for (int n : {INT_MIN, -1, 0, 1, 2, 31, 32, 33, 255, 256, 257, INT_MAX}) {
        const LatentRecord r{v, n};
        if (latent_record_joins(r, side))
          for (int j = 0; j < n; ++j)
            CHECK(latent_record_slot(r, side, j) >= 0 && latent_record_slot(r, side, j) < 2 * kLatentUnits);
      }
  for (int k = 0; k < 200; ++k) {  // equal lengths, some of which fit the shares
    const int B = 1 << pick(0, 8), n = pick(1, 4);
    std::vector<int> cu{0}, lens(B, 64 * pick(1, 60));
    for (int b = 0; b < B; ++b) cu.push_back(cu.back() + n);
    walk(cu, lens, cu.back(), 16, 16 << pick(0, 2), 1 << pick(0, 3), 1 << 16, 2);
  }
  CHECK(whole > 20 && cut > 100);
  std::printf("%lld walked, %lld violations\n", walked, bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_every_work_group_of_every_batch(tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(WALKER)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}", str(src), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.endswith(" 0 violations\n")
