"""CPU: how one launch deals its work-groups to the shared prefixes and the sequences' own keys
(csrc/latent_plan.hpp): every step of both lines is taken once, whole tiles have blocks of their own."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "latent_plan.hpp"
using namespace ferret;

static int line(const std::vector<LatentSeq>& seqs, int units, int side, int min_steps) {
  int all = 0, groups = 0;
  for (const auto& s : seqs) all = latent_add(all, s.work(0)), groups = latent_add(groups, s.groups);
  bool whole = true;
  for (const auto& s : seqs) whole = whole && latent_fits(s, latent_chunk(all, units, min_steps));
  const LatentDeal d = latent_deal(all, groups, whole, units, min_steps);
  if ((long long)d.chunk * units < d.total) return 1;  // the units take the whole line
  int at = 0;
  for (const auto& s : seqs)
    for (int g = 0; g < s.groups; ++g, at += s.steps + d.extra) {
      const int unit = at / d.chunk;
      if (unit >= units) return 2;
      const LatentRecord r = latent_record(unit, 0, side, at, s.steps, d.chunk);
      if (r.pieces > 1 && !latent_record_joins(r, side)) return 3;
      for (int j = 0; j < r.pieces; ++j)
        if (r.pieces > 1 && latent_record_slot(r, side, j) >= 2 * units * side) return 4;
    }
  return 0;
}

int main() {
  std::srand(11);
  // the deal itself
  for (int i = 0; i < 200000; ++i) {
    const int first = std::rand() % 5 == 0 ? 0 : std::rand() >> (std::rand() % 31), second = std::rand() % 5 == 0 ? 0 : std::rand() >> (std::rand() % 31);
    const int s0 = 1 + std::rand() % 2, s1 = 1 + std::rand() % 2, g = latent_split(first, second, 0.5f + std::rand() % 4, s0, s1);
    if (g < 0 || g > kLatentUnits || g % (8 * s0) || (kLatentUnits - g) % (8 * s1)) return std::printf("groups %d\n", g), 1;
    if ((first > 0 && g == 0) || (second > 0 && g == kLatentUnits) || (first == 0 && g != 0)) return std::printf("starved\n"), 1;
    for (int b = 0; b < kLatentUnits; ++b) {
      const bool mine = b < g;
      const LatentPlace p = latent_place(mine ? b : b - g, mine ? s0 : s1);
      if (p.unit < 0 || p.unit >= (mine ? g / s0 : (kLatentUnits - g) / s1) || p.lane < 0 || p.lane >= (mine ? s0 : s1) ||
          p.unit % 8 != b % 8)
        return std::printf("place\n"), 1;
    }
  }
  // lines of many batches on few and many units; blocks of whole tiles
  for (int i = 0; i < 3000; ++i) {
    const int H = 1 + std::rand() % 130, B = 1 + std::rand() % 40, mr = 16 << std::rand() % 3, side = 1 + std::rand() % 2;
    int T = 0;
    std::vector<int> n(B), len(B);
    for (int b = 0; b < B; ++b) {
      n[b] = std::rand() % 3 == 0 ? 0 : std::rand() % 2 ? 1 : std::rand() % 60;
      len[b] = std::rand() % 4 == 0 ? 0 : std::rand() % 9000;
      T += n[b];
    }
    if (T == 0) continue;
    std::vector<LatentSeq> seqs;
    const int blocks = T * H / 16 + B + 4;
    std::vector<int> taken(blocks, 0);
    int q0 = 0;
    for (int b = 0; b < B; q0 += n[b++]) {
      seqs.push_back(latent_seq(q0, q0 + n[b], len[b], T, H, mr, side, 1 << 30));
      const int rows = n[b] * H;
      for (int row0 = 0; row0 < rows; row0 += 16) {
        const int at = (q0 * H >> 4) + b + (row0 >> 4);
        if (at >= blocks || taken[at]++) return std::printf("block %d\n", at), 1;
      }
    }
    for (int units : {8, 16, 24, 128, 256})
      if (units % (8 * side) == 0 || side == 1)
        if (units * side <= kLatentUnits)
          if (const int rc = line(seqs, units, side, mr == 64 ? 2 : 1)) return std::printf("line %d\n", rc), 1;
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_two_lines_in_one_launch(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


SEARCH = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "latent_plan.hpp"
using namespace ferret;
int main() {
  std::srand(12);
  for (int i = 0; i < 20000; ++i) {
    const int G = 1 + std::rand() % 12;
    std::vector<int> starts(G + 1);
    starts[0] = std::rand() % 5;
    for (int g = 0; g < G; ++g) starts[g + 1] = starts[g] + (std::rand() % 3 == 0 ? 0 : std::rand() % 9);
    for (int q = 0; q <= starts[G] + 2; ++q) {
      int want = -1;
      for (int g = 0; g < G; ++g)
        if (starts[g] <= q && q < starts[g + 1]) want = g;
      if (latent_prefix(starts.data(), G, q) != want) return std::printf("token %d\n", q), 1;
    }
    for (int& x : starts) x = std::rand() - std::rand();  // whatever stands there, a line of the table
    for (int q = 0; q < 50; ++q) {
      const int g = latent_prefix(starts.data(), G, std::rand() % 1000);
      if (g < -1 || g >= G) return std::printf("line %d\n", g), 1;
    }
  }
  // own keys behind a prefix's: on the next whole step, nothing lost
  for (int prefix = 0; prefix < 400; ++prefix)
    for (int len = 0; len < 200; ++len) {
      LatentSeq s = latent_seq(0, 1, len, 1, 16, 16, 1, 1 << 20);
      latent_behind(&s, prefix);
      const int base = latent_base(prefix);
      if (base < prefix || base >= prefix + kLatentKeys || base % kLatentKeys || s.len != base + len) return std::printf("base\n"), 1;
      if (s.steps < 1 || s.steps * kLatentKeys < s.len || (s.steps > 1 && (s.steps - 1) * kLatentKeys >= s.len)) return std::printf("steps\n"), 1;
    }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_the_prefix_of_a_sequence(tmp_path):
    src, exe = tmp_path / "search.cpp", tmp_path / "search"
    src.write_text(SEARCH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
