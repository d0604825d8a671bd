"""CPU: which rows a join hands to work-groups of their own (csrc/latent_plan.hpp).  What a row has in pieces follows
from the lengths on the device; the host knows the mean alone, and one long sequence among short ones has many
times that."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <vector>
#include "latent_plan.hpp"
using namespace ferret;

static int worst = 0;

// The tiles of more than `few` pieces are those that the work-groups note, each by the one that begins it.
static int walk(const std::vector<int>& n, const std::vector<int>& lens, int H, int mr, int side, int most, int min_steps) {
  std::vector<LatentSeq> seqs;
  int T = 0, q0 = 0, all = 0, groups = 0;
  for (int x : n) T += x;
  for (size_t b = 0; b < n.size(); q0 += n[b++]) {
    seqs.push_back(latent_seq(q0, q0 + n[b], lens[b], T, H, mr, side, most));
    all = latent_add(all, seqs.back().work(0)), groups = latent_add(groups, seqs.back().groups);
  }
  const int units = kLatentUnits / side;
  bool whole = true;
  for (const auto& s : seqs) whole = whole && latent_fits(s, latent_chunk(all, units, min_steps));
  const LatentDeal d = latent_deal(all, groups, whole, units, min_steps);
  const long long rows = (long long)T * H, steps = most / kLatentKeys + 1;
  long long mean = (long long)kLatentUnits * mr / rows, top = kLatentUnits / side;
  if (steps < mean) mean = steps;
  if (steps < top) top = steps;
  const LatentJoin j = latent_join(mean, top, rows, false);
  std::set<int> want, got;
  int at = 0, longest = 0;
  for (const auto& s : seqs)
    for (int g = 0; g < s.groups; ++g, at += s.steps + d.extra) {
      const int unit = at / d.chunk, pieces = latent_record(unit, 0, side, at, s.steps, d.chunk).pieces;
      if (pieces > longest) longest = pieces;
      for (int lane = 0; lane < side; ++lane)
        if ((g * side + lane) * mr < s.rows && pieces > j.few) want.insert(s.q0 * H + (g * side + lane) * mr);
    }
  for (int block = 0; block < kLatentUnits; ++block) {
    const LatentPlace p = latent_place(block, side);
    const int start = plan_min((int)plan_min(p.unit * d.chunk, d.total), d.total), end = plan_min(start + d.chunk, d.total);
    if (start >= d.total) continue;
    int b = 0, seq_at = 0;
    while (seq_at + seqs[b].work(d.extra) <= end - 1) seq_at += seqs[b++].work(d.extra);
    const int row = latent_many(seqs[b], seq_at, d.extra, end, d.chunk, side, p.lane, mr, H, j.few);
    if (row >= 0 && !got.insert(row).second) return 1;
  }
  if (want != got) return 2;
  // what one wave or group of waves takes one after another
  if (longest > top) return 3;
  const int left = longest > j.few ? j.few : longest;
  const int by_units = (left + latent_join_ahead(j.waves) - 1) / latent_join_ahead(j.waves);
  const int by_many = longest > j.few ? (longest + latent_join_ahead(kLatentManyWaves) - 1) / latent_join_ahead(kLatentManyWaves) : 0;
  for (int r : {by_units, by_many})
    if (r > worst) worst = r;
  return 0;
}

int main() {
  std::srand(5);
  const auto pick = [](int lo, int hi) { return lo + std::rand() % (hi - lo + 1); };
  for (int i = 0; i < 4000; ++i) {
    const int B = pick(1, 90), H = 1 << pick(0, 7), mr = 16 << pick(0, 2), side = 1 << pick(0, 3), most = 64 << pick(0, 11);
    std::vector<int> n(B), lens(B);
    for (int b = 0; b < B; ++b) {
      n[b] = pick(0, 6) ? 1 : pick(0, 40);
      lens[b] = i % 2 ? pick(0, most) : pick(0, 200);
    }
    n[pick(0, B - 1)] = 1;
    if (i % 2 == 0) lens[pick(0, B - 1)] = most;  // one long among short ones
    if (const int rc = walk(n, lens, H, mr, side, most, mr == 64 ? 2 : 1)) return std::printf("batch %d: %d\n", i, rc), 1;
  }
  // 16 heads, one token each: one sequence of 100001 keys among others of 100
  for (int B = 1; B <= 600; ++B) {
    std::vector<int> n(B, 1), lens(B, 100);
    lens[B / 2] = 100001;
    if (const int rc = walk(n, lens, 16, 16, 1, 100032, 1)) return std::printf("skewed %d: %d\n", B, rc), 1;
  }
  std::printf("%d rounds at most\n", worst);
  return worst > 12;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_no_row_is_joined_piece_after_piece(tmp_path):
    """By the mean alone a wave would take 224 pieces of the one long sequence four at a time: 56 rounds."""
    src, exe = tmp_path / "join.cpp", tmp_path / "join"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_waves_of_few_and_of_many_rows(tmp_path):
    """Eight and sixteen waves to 16 rows only where the rows leave room for them: 648 rows of 25 pieces took 31.0 us with
    eight and 27.3 with four, 32 rows of 128 20.5 with eight and 19.6 with sixteen."""
    src, exe = tmp_path / "waves.cpp", tmp_path / "waves"
    src.write_text('#include <cstdio>\n#include "latent_plan.hpp"\nint main() { const long long at[][2] = {{25, 648}, {128, 32}, {64, '
                   '64}, {48, 128}, {48, 129}, {32, 512}, {24, 513}, {16, 256}, {8, 512}, {1, 16000}};\nfor (const auto& a : at) '
                   'std::printf("%d ", ferret::latent_join(a[0], 256, a[1], false).waves); }\n')
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == [4, 16, 16, 16, 8, 8, 4, 4, 1, 1]
