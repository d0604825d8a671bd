// The order in which the expanded attention takes its query tiles.  Plain C++17 without
// HIP, so that a CPU test compiles it on its own and checks that every tile of a ragged
// batch is taken once, the longest first (tests/test_expanded_plan.py).
#pragma once

#ifdef __HIPCC__
#define FERRET_XHD __host__ __device__ __forceinline__
#else
#define FERRET_XHD inline
#endif

namespace ferret {

constexpr int kTileTokens = 128;   // query tokens per tile
constexpr int kTileKeys = 64;      // keys per step
// Sequences up to which tiles go by length over the whole batch: the search costs each
// work-group about 0.15 us per sequence.  By length / sequence by sequence, 16 heads, us: four
// prompts of 700 to 1900 63.2 / 67.9, eight of 300 to 1300 63.7 / 71.3, sixteen of 100 to 700
// 59.9 / 55.3, forty of 50 to 300 94.6 / 49.7.
constexpr int kOrderedBatch = 8;

// The tiles of one sequence: n new tokens, the last of len keys.
struct TileSeq {
  int n, len, causal;
  FERRET_XHD int tiles() const { return (n + kTileTokens - 1) / kTileTokens; }
  // The first tile of at least `steps` steps (tiles() for none): a tile's steps grow
  // with its number, by two from one to the next.
  FERRET_XHD int first_of(int steps) const {
    const int t = tiles();
    if (steps <= 0) return 0;
    const int keys = kTileKeys * (steps - 1) + 1;  // that the tile's last token has to see
    if (t == 0 || len < keys) return t;
    if (!causal) return 0;
    const int rows = keys - (len - n);  // the tile's end has to reach this row
    const int at = rows <= 0 ? 0 : (rows + kTileTokens - 1) / kTileTokens - 1;
    return at < t - 1 ? at : t - 1;
  }
  FERRET_XHD int at_least(int steps) const { return tiles() - first_of(steps); }
};

// Where two work-groups share a CU, the second `first` slots of a head (a CU's worth each)
// go from short to long, so that the longest tiles do not meet the next longest (4096
// tokens after 4096 others, 16 heads: 240 us, 257 without).
FERRET_XHD int paired_rank(int slot, int all, int first) {
  const int both = all < 2 * first ? all : 2 * first;
  return slot < first || slot >= both ? slot : both - 1 - (slot - first);
}

}  // namespace ferret
