// Launch plan and arguments of the int8 product (int8_gemm.hip).  Plain C++17
// without HIP, so that a CPU test walks it over shapes.
#pragma once

#include <cstddef>
#include <cstdint>

namespace ferret {
namespace i8 {

struct Args {
  const uint8_t* a;          // int8 tokens [M, K]
  const float* sa;           // [M]
  const uint8_t* b;          // int8 weights [N, K]
  const float* sb;           // [N]
  const uint16_t* residual;  // bf16 [M, N] or null
  uint16_t* out;             // bf16 [M, N]
  int32_t* partial;          // splits > 1: [splits, M, N]
  int M, N, K;
  int splits;                // K splits
  int tok_tiles;             // token tiles
  bool nt;                   // stream the weights past the caches
};

// The tiles the kernel is built for: rt x 16 weight rows by tt x 16 tokens, ks
// bytes of K per stage, ns stages in LDS.
struct Tile {
  int rt, tt, ks, ns;
};
constexpr Tile kTiles[] = {
    {4, 1, 256, 4}, {6, 1, 256, 5}, {4, 2, 256, 5}, {6, 2, 256, 5}, {4, 4, 256, 4}, {6, 4, 256, 4},
    {4, 8, 256, 3}, {8, 8, 128, 4}};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);

constexpr int kMostSplits = 8;

struct Plan {
  int tile = 0;
  int splits = 1;
  int tok_tiles = 1;
};

inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

// The tile and K split with the least estimated time.
inline Plan plan(int M, int N, int K, int ncu) {
  Plan best;
  double best_t = -1;
  for (int i = 0; i < kNumTiles; ++i) {
    const Tile& t = kTiles[i];
    const long long tok_tiles = cdiv(M, 16 * t.tt), tiles = tok_tiles * cdiv(N, 16 * t.rt);
    if (tok_tiles > 1 && t.tt < 8) continue;
    const double wb = t.rt * 16.0 * t.ks, xb = t.tt * 16.0 * t.ks;  // bytes of a stage
    const double stage_w = wb / 25e3, stage_all = (wb + xb) / 46e3;
    const double stage = stage_w > stage_all ? stage_w : stage_all;  // us
    for (int s = 1; s <= kMostSplits; ++s) {
      if (s > 1 && (M > 2048 || tiles >= 2LL * ncu)) break;
      const long long steps = cdiv(cdiv(K, t.ks), s), rounds = cdiv(tiles * s, ncu);
      const double us = rounds * (steps * stage + 1.5) + (s > 1 ? 3.0 + (double)s * M * N * 8 / 4e6 : 0.0);
      if (tiles * s < (1LL << 31) && (best_t < 0 || us < best_t)) {
        best_t = us;
        best.tile = i;
        best.splits = s;
        best.tok_tiles = (int)tok_tiles;
      }
    }
  }
  return best;
}

}  // namespace i8
}  // namespace ferret
