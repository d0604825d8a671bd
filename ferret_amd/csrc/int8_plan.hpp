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

// A tile that a kernel is built for: rows of weights by tokens, ks bytes of K per stage,
// and what it takes of a CU, us: start once, then per round of work-groups `round` and
// per stage `stage`; rate: the TB/s at which it streams bytes.
struct Tile {
  int rows, toks, ks;
  float start, round, stage, rate;
};
constexpr Tile kTiles[] = {
    // int8_gemm.hip: all tokens in one tile
    {16, 16, 512, 2.7f, 0.4f, 0.33f, 5.8f},
    {32, 16, 256, 3.0f, 0.05f, 0.28f, 6.0f},
    {96, 16, 256, 2.6f, 1.1f, 0.50f, 6.2f},
    {32, 32, 512, 1.0f, 2.3f, 0.58f, 5.9f},
    {96, 64, 256, 3.0f, 1.3f, 0.74f, 6.0f},
    // int8_square.hip
    {64, 32, 256, 3.8f, 0.35f, 0.35f, 5.8f},
    {64, 64, 128, 3.3f, 0.6f, 0.23f, 5.8f},
    {64, 128, 128, 3.3f, 1.3f, 0.31f, 5.8f},
    {128, 128, 128, 1.0f, 4.1f, 0.49f, 5.8f},  // eight waves
    {128, 128, 128, 5.1f, 1.5f, 0.50f, 5.8f},  // four, two work-groups per CU
    {256, 128, 128, 1.0f, 6.0f, 0.75f, 5.8f},
    {256, 256, 128, 1.0f, 9.2f, 1.30f, 5.8f}};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]), kFirstSquare = 5;
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8};
constexpr int kCus = 256;

struct Plan {
  int tile = -1;
  int splits = 1;
  int tok_tiles = 1;
};

inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

// The tile and K split with the least expected time: what the fullest CU's work-groups
// take one after another, or the bytes at its rate; a split adds its sum's launch and the
// partials' way out and back.  The tiles' figures are fits to the times of 240 shapes (1
// to 8192 tokens, 512 to 24576 rows, K from 512 to 12288): their choice takes 1.1% longer
// than the best of all tiles and splits that were timed (geometric mean; 7% in 95 of 100).
// Both sides, us: 4096 x 4096 at 16 tokens 6.3 of 16 x 16, 7.0 of 32 x 16; 24576 x 4096
// at 16 17.4 of 96 x 16, 20.2 of 32 x 16; 7168 x 2048 at 100 8.4 of 64 x 64, 9.9 of 64 x 128;
// 4096 x 7168 at 100 14.4 of 64 x 128 in 4 splits, 17.9 of 64 x 64 in one; 6144 x 4096 at
// 1000 29.9 of 256 x 128, 32.1 of 128 x 128; 4096 x 7168 at 4096 102 of 256 x 256, 115 of 256 x 128.
inline Plan plan(int M, int N, int K) {
  Plan best;
  double best_t = 0;
  const double mn = (double)M * N, bytes = (double)M * K + (double)N * K + 2 * mn;
  for (int i = 0; i < kNumTiles; ++i) {
    const Tile& t = kTiles[i];
    const long long tok_tiles = cdiv(M, t.toks), tiles = tok_tiles * cdiv(N, t.rows), stages = cdiv(K, t.ks);
    if (tok_tiles > 1 && i < kFirstSquare) continue;
    const double stream = bytes / (t.rate * 1e6) + 2.0;
    for (const int s : kSplits) {
      if (s > 1 && (s > stages || tiles * s > 4 * kCus)) break;
      const double cu = t.start + (double)cdiv(tiles * s, kCus) * (t.round + (double)cdiv(stages, s) * t.stage);
      const double us = (cu > stream ? cu : stream) + (s > 1 ? 3.0 + s * mn * 8 / 5e6 : 0.0);
      if (best.tile < 0 || us < best_t) {
        best_t = us;
        best.tile = i;
        best.splits = s;
        best.tok_tiles = (int)tok_tiles;
      }
    }
  }
  return best;
}

// Bytes of the partial sums of a plan.
inline size_t workspace(const Plan& plan, int M, int N) {
  return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(int32_t) : 0;
}

}  // namespace i8
}  // namespace ferret
