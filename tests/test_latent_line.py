"""CPU: the latent attention's line of steps where sequences overlap in a batch whose starts do not ascend.

The sequences' works then add up past 32 bits although each is within them.  Compiles
ferret_amd/csrc/latent_plan.hpp with g++ and follows how a work-group of latent_attention.hip adds up its
threads' sequences and finds its share: either nobody gets a share, or exactly one thread names each one.
"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ferret_amd", "csrc")

WALKER = r"""
#include <climits>
#include <cstdio>
#include <vector>
#include "latent_plan.hpp"
using namespace ferret;

static long long bad = 0, none = 0, dealt = 0;
#define CHECK(c) do { if (!(c) && bad++ < 20) std::printf("line %d: %s\n", __LINE__, #c); } while (0)

static void share(int B, int T, int H, int mr, int side, int most, int threads) {
  const int units = kLatentUnits / side, per = (B + threads - 1) / threads;
  std::vector<int> cu;
  for (int b = 0; b <= B; ++b) cu.push_back(b % 2 ? T : 0);
  std::vector<int> incl(threads), incl_groups(threads), mine(threads), my_groups(threads);
  long long exact = 0, exact_groups = 0;
  int total = 0, groups = 0;
  bool fits = per == 1;
  for (int t = 0; t < threads; ++t) {
    for (int i = 0; i < per && t * per + i < B; ++i) {
      const LatentSeq s = latent_seq(cu[t * per + i], cu[t * per + i + 1], most, T, H, mr, side, most);
      mine[t] = latent_add(mine[t], s.work(0));
      my_groups[t] = latent_add(my_groups[t], s.groups);
      exact += s.work(0);
      exact_groups += s.groups;
    }
    incl[t] = total = latent_add(total, mine[t]);
    incl_groups[t] = groups = latent_add(groups, my_groups[t]);
  }
  CHECK(total == (exact < INT_MAX ? exact : INT_MAX) && groups == (exact_groups < INT_MAX ? exact_groups : INT_MAX));
  for (int b = 0; b < B; ++b)
    fits = fits && latent_fits(latent_seq(cu[b], cu[b + 1], most, T, H, mr, side, most), latent_chunk(total, units, 1));
  const LatentDeal d = latent_deal(total, groups, fits, units, 1);
  const long long line = exact + (fits ? 0 : kLatentExtra * exact_groups);
  if (line > INT_MAX - kLatentUnits) {
    CHECK(d.total == 0);
    ++none;
    return;
  }
  CHECK(d.total == line && d.chunk >= 1 && (long long)d.chunk * units >= line);
  ++dealt;
  for (int unit = 0; unit < units; ++unit) {
    if ((long long)unit * d.chunk >= d.total) continue;
    const int start = unit * d.chunk;
    int named = 0;
    for (int t = 0; t < threads; ++t) {
      const int excl = incl[t] - mine[t] + d.extra * (incl_groups[t] - my_groups[t]);
      named += excl <= start && start < excl + mine[t] + d.extra * my_groups[t];
    }
    CHECK(named == 1 && start + d.chunk > start);
  }
}

int main() {
  for (int threads : {256, 512})
    for (int B : {1, 2, 7, 64, 255, 256, 257, 700, 3000})
      for (int side : {1, 8})
        for (int mr : {16, 64})
          for (int T : {1, 100, 4096})
            for (int most : {16, 1000, 1 << 20, 1 << 24}) {
              const long long tiles = (long long)T * 128 / mr + B, steps = ((long long)most + 63) / 64 + kLatentExtra;
              if (tiles * steps < (1LL << 31) - kLatentUnits) share(B, T, 128, mr, side, most, threads);
            }
  CHECK(none > 50 && dealt > 200);
  std::printf("%lld without, %lld dealt, %lld violations\n", none, dealt, bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_a_share_is_named_once_or_there_is_none(tmp_path):
    src = tmp_path / "line.cpp"
    src.write_text(WALKER)
    exe = tmp_path / "line"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}",
                    str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.endswith(" 0 violations\n")


NEAR = r"""
#include <climits>
#include <cstdio>
#include <initializer_list>
#include "latent_plan.hpp"
using namespace ferret;
int main() {
  long long bad = 0;
  for (int units : {32, 64, 128, 256})
    for (int B : {1, 2, 31, 32, 33, 255, 256, 257, 600, 8421504, 8421505, 9000000, 1 << 28, INT_MAX})
      for (int unit = 0; unit < units; ++unit) bad += latent_near(unit, units, B) != (long long)unit * B / units;
  std::printf("%lld off\n", bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_the_sequence_looked_up_first_is_one_of_the_batch(tmp_path):
    """Also where unit * B passes 32 bits (from 8421505 sequences on)."""
    src = tmp_path / "near.cpp"
    src.write_text(NEAR)
    exe = tmp_path / "near"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}",
                    str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr
