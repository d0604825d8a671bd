"""CPU: the launch plan of the int8 product (csrc/int8_plan.hpp) walked over shapes: every plan is one that the
kernels are built for, its splits all have stages, and the tiles that no shape would reach are none."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "int8_plan.hpp"
using namespace ferret::i8;
int main() {
  int seen[kNumTiles] = {0};
  bool split[9] = {false};
  const int Ns[] = {8, 16, 72, 264, 512, 1000, 2048, 4096, 6144, 7168, 12000, 16384, 24576, 153600, 1 << 20};
  const int Ks[] = {16, 48, 128, 512, 528, 1040, 2048, 4096, 7168, 12288, 65536};
  long long n = 0;
  for (int N : Ns)
    for (int K : Ks)
      for (long long M = 1; M <= 70000; M += M < 140 ? 1 : M / 9) {
        const Plan p = plan((int)M, N, K);
        if (p.tile < 0 || p.tile >= kNumTiles) return std::printf("tile %d at %lld %d %d\n", p.tile, M, N, K), 1;
        const Tile& t = kTiles[p.tile];
        const long long tiles = cdiv(N, t.rows) * p.tok_tiles * p.splits;
        if (p.tok_tiles != cdiv(M, t.toks) || (p.tile < kFirstSquare && p.tok_tiles != 1) || tiles >= (1LL << 31) ||
            p.splits < 1 || p.splits > 8 || (p.splits > 1 && p.splits > cdiv(K, t.ks)))
          return std::printf("plan %d x%d at %lld %d %d\n", p.tile, p.splits, M, N, K), 1;
        // every split has a stage, and together they have all of them
        const long long stages = cdiv(K, t.ks);
        long long sum = 0;
        for (int s = 0; s < p.splits; ++s) {
          const long long k0 = s * stages / p.splits, k1 = (s + 1) * stages / p.splits;
          if (k1 <= k0) return std::printf("empty split at %lld %d %d\n", M, N, K), 1;
          sum += k1 - k0;
        }
        if (sum != stages || workspace(p, (int)M, N) != (p.splits > 1 ? 4ull * p.splits * M * N : 0)) return 1;
        seen[p.tile]++;
        split[p.splits] = true;
        ++n;
      }
  for (int i = 0; i < kNumTiles; ++i)
    if (seen[i] == 0) return std::printf("tile %d is never chosen\n", i), 1;
  for (int s : kSplits)
    if (!split[s]) return std::printf("%d splits are never chosen\n", s), 1;
  std::printf("%lld plans\n", n);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_every_plan_can_run(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_gpu_shapes_reach_every_tile(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not installed")
    import ast
    text = open(os.path.join(ROOT, "tests", "test_gpu_int8.py")).read()
    at = text.index("TILES = ") + len("TILES = ")
    shapes = ast.literal_eval(text[at:text.index("]\n", at) + 1])
    src, exe = tmp_path / "tiles.cpp", tmp_path / "tiles"
    src.write_text('#include <cstdio>\n#include "int8_plan.hpp"\nint main() { int m, n, k; while (std::scanf("%d %d %d", &m, '
                   '&n, &k) == 3) { auto p = ferret::i8::plan(m, n, k); std::printf("%d %d\\n", p.tile, p.splits); }\n'
                   'std::printf("%d 0\\n", ferret::i8::kNumTiles); }\n')
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/ferret_amd/csrc", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], input="\n".join("%d %d %d" % s for s in shapes), capture_output=True, text=True).stdout
    *plans, (tiles, _) = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert {t for t, _ in plans} == set(range(tiles))
    assert {t for t, s in plans if s > 1} >= {0, 1, 2, 3, 4, 5, 6, 7, 8}
