// How the latent attention deals a ragged batch to its work-groups, and where a
// position's row stands in the paged cache.  Plain C++17 without HIP, so that a CPU
// test compiles it on its own and walks every work-group of many batches
// (tests/test_latent_plan.py): every (sequence, row tile, step) is taken once, no two
// pieces share a slot, the records lead to exactly the pieces of a tile, and no row
// outside the cache is named, whatever the index tensors hold.
#pragma once

#include <climits>

#ifdef __HIPCC__
#define FERRET_HD __host__ __device__ __forceinline__
#else
#define FERRET_HD inline
#endif

namespace ferret {

constexpr int kLatentKeys = 64;    // keys per step
constexpr int kLatentUnits = 256;  // work-groups the work is dealt to: one per CU
constexpr int kLatentExtra = 5;    // steps that going from one tile to the next costs

FERRET_HD int plan_min(int a, int b) { return a < b ? a : b; }
FERRET_HD int plan_max(int a, int b) { return a > b ? a : b; }

// The row of `offset` in page `id`, -1 where id names no page.
FERRET_HD long long page_row(int id, int pages, int page_size, int offset) {
  return (unsigned)id < (unsigned)pages ? (long long)id * page_size + offset : -1;
}

// The work of one sequence: query rows (token-major, then heads) in tiles of `mr`,
// `side` of which are taken side by side (each by a work-group of its own, over the
// same keys at the same time) as one group; keys in steps.  Index values outside the
// tensors are cut to them.
struct LatentSeq {
  int q0, n, len, rows, groups, steps;
  FERRET_HD int work(int extra) const { return groups * (steps + extra); }
};

FERRET_HD LatentSeq latent_seq(int start, int end, int len, int T, int H, int mr, int side, int most_keys) {
  LatentSeq s;
  s.q0 = plan_min(plan_max(start, 0), T);
  s.n = plan_min(plan_max(end, s.q0), T) - s.q0;
  s.len = plan_min(plan_max(len, 0), most_keys);
  s.rows = s.n * H;
  s.groups = (s.rows + mr * side - 1) / (mr * side);
  s.steps = plan_max((s.len + kLatentKeys - 1) / kLatentKeys, 1);  // an empty sequence's rows are written too
  return s;
}

// A sequence whose own keys stand behind those of a prefix: on the next whole step, so that no
// step has keys of both.
FERRET_HD int latent_base(int prefix) { return (prefix + kLatentKeys - 1) / kLatentKeys * kLatentKeys; }
FERRET_HD void latent_behind(LatentSeq* s, int prefix) {
  s->len += latent_base(prefix);
  s->steps = plan_max((s->len + kLatentKeys - 1) / kLatentKeys, 1);
}

// The prefix whose tokens, starts[g] .. starts[g + 1] - 1, hold q0; -1 where none does.
FERRET_HD int latent_prefix(const int* starts, int prefixes, int q0) {
  int at = 0, end = prefixes;  // the last of at .. end - 1 that starts at q0 or before
  while (end - at > 1) {
    const int half = at + (end - at) / 2;
    if (starts[half] <= q0) at = half;
    else end = half;
  }
  return starts[0] <= q0 && q0 < starts[prefixes] ? at : -1;
}

// The line of all (sequence, group, step) is dealt in equal shares to `units` =
// kLatentUnits / side units of `side` work-groups.  Each group is followed by `extra`
// steps without keys, so that a unit that goes on to a second tile (its queries, and the
// first keys' way from memory) is not the last to end: kLatentExtra, or none where
// every sequence is a whole number of shares as it is (latent_fits).  16 rows, e4m3, 64
// sequences of 600 to 8000 keys: 55.5 us without, 50.4 with 5; 64 rows, bf16, 32 of
// 2000: 42.3 us without, 46.8 with 5.  Steps per unit of a line of `total`:
FERRET_HD int latent_chunk(int total, int units, int min_steps) {
  return plan_max(min_steps, total / units + (total % units != 0));
}

FERRET_HD bool latent_fits(const LatentSeq& s, int chunk) { return s.groups == 0 || s.steps % chunk == 0; }

// Sums of work along the line, of numbers from 0 on; they stop at INT_MAX.  Starts that ascend
// stay far below it (the caller checks T and the table's keys); where they do not, sequences
// overlap, and a sum that went round would lead to shares that nobody or several name.
FERRET_HD int latent_add(int a, int b) {
  const unsigned sum = (unsigned)a + (unsigned)b;
  return sum > (unsigned)INT_MAX ? INT_MAX : (int)sum;
}

// The deal of a line of `total` steps in `groups` groups to `units` units: total 0 where
// there is nothing to do, or where it does not fit 32 bits.
struct LatentDeal {
  int total, chunk, extra;
};
FERRET_HD LatentDeal latent_deal(int total, int groups, bool fits, int units, int min_steps) {
  const int extra = fits ? 0 : kLatentExtra;
  const long long line = total + (long long)extra * groups;
  if (line > INT_MAX - kLatentUnits) return LatentDeal{0, 1, 0};
  return LatentDeal{(int)line, latent_chunk((int)line, units, min_steps), extra};
}

// The unit and the place in it of a work-group.  Work-groups are dealt to the 8 XCDs
// in turn; a unit's stay on one, so that its keys come from memory once.
struct LatentPlace {
  int unit, lane;
};
FERRET_HD LatentPlace latent_place(int block, int side) {
  return LatentPlace{block / (8 * side) * 8 + block % 8, block / 8 % side};
}

// Work-groups of kLatentUnits for the first of two lines of steps that one launch takes, each
// dealt to units of its own, `side` work-groups to a unit: in proportion to the steps, one of the first
// line's as long as `weight` of the second's; whole rounds of 8 units, so that a unit's
// work-groups stay on one XCD; some for each line that has steps.
FERRET_HD int latent_split(int first, int second, float weight, int first_side, int second_side) {
  const int round = 8 * plan_max(first_side, second_side);
  if (first == 0) return 0;
  if (second == 0) return kLatentUnits;
  const float a = weight * (float)first, share = a / (a + (float)second);
  const int rounds = (int)(share * (float)(kLatentUnits / round) + 0.5f);
  return round * plan_min(plan_max(rounds, 1), kLatentUnits / round - 1);
}

// A sequence that a unit's share may start in, were all alike: floor(unit * B / units),
// without the product, which passes 32 bits from 2^23 sequences on.
FERRET_HD int latent_near(int unit, int units, int B) { return unit * (B / units) + unit * (B % units) / units; }

// The slot of the partial result that a unit's work-group takes up at `cur` of the
// line: the share may start and end inside a tile, so there are two each.
FERRET_HD int latent_slot(int unit, int lane, int side, int cur, int chunk) {
  return 2 * (unit * side + lane) + (cur > unit * chunk ? 1 : 0);
}

// Where the pieces of a tile of `steps` steps stand that `unit` begins at `cur`: the first in its slot
// `odd`, the others each in the even slot of the next unit.  slot0 is the first's.
struct LatentRecord {
  int slot0, pieces;
};
FERRET_HD LatentRecord latent_record(int unit, int lane, int side, int cur, int steps, int chunk) {
  return LatentRecord{latent_slot(unit, lane, side, cur, chunk), (cur + steps - 1) / chunk - unit + 1};
}
FERRET_HD int latent_record_slot(const LatentRecord& r, int side, int piece) {
  return piece == 0 ? r.slot0 : (r.slot0 & ~1) + 2 * side * piece;
}
// The first row, among all, of the tile of more than `few` pieces that a work-group begins, -1
// where it begins none: the tile is the last of its share, which ends at `end` of the line, in
// sequence `s`, at `seq_at`, and takes all of the next shares but the last of its own.
FERRET_HD int latent_many(const LatentSeq& s, int seq_at, int extra, int end, int chunk, int side, int lane, int mr,
                          int H, int few) {
  const long long whole = (long long)(few - 1) * chunk;
  if (s.steps <= whole) return -1;
  const int group = (end - 1 - seq_at) / (s.steps + extra), at = seq_at + group * (s.steps + extra);
  const int row0 = (group * side + lane) * mr;
  const bool many = group < s.groups && at >= end - chunk && s.steps > end - at + whole;
  return many && row0 < s.rows ? s.q0 * H + row0 : -1;
}
// More than one piece, all of them inside the workspace (a row that no sequence
// covers has no record, and whatever stands there must lead nowhere else).
FERRET_HD bool latent_record_joins(const LatentRecord& r, int side) {
  return r.pieces >= 2 && r.pieces <= kLatentUnits && (unsigned)r.slot0 < (unsigned)(2 * kLatentUnits) &&
         (r.slot0 | 1) + 2 * side * (r.pieces - 1) < 2 * kLatentUnits;
}

// How the pieces of `rows` rows are joined: by `waves` waves to 16 rows, which take
// latent_join_ahead() pieces at a time together, but rows of more than `few` pieces by work-groups of
// kLatentManyWaves waves.  mean: a row's pieces on average, all work-groups at the rows
// there are; most: where one sequence has nearly all of the keys.  Us, whole call, with 1 / 4 / 8 /
// 16 waves: 16 heads, e4m3, one sequence of 100001 (256 pieces) - / - / 29.7 / 28.0; bf16, two of 2863 and 10431 (128)
// - / - / 20.5 / 19.6; 128 heads, four of 9831 (512 rows, 32 pieces) - / 34.2 / 34.1 / 38.9; chunks of 27 and 54 tokens,
// 8 heads (648 rows, 25) - / 27.3 / 31.0 / -; 64 sequences behind 8192 keys (16 + 4) 50.7 / 49.2 / - / 58.5.  Every row alike / as
// here: rows that can have 32 pieces at most (chunks of 200 to 500 tokens) 168.9, with few 12 175.4; two passes, of
// which a row has pieces of both, 128 sequences behind 4096 55.3, with few 48 57.8; 256 behind 4096 (5 pieces on
// average) 73.6 / 74.5, with one of 120000 own keys 97.7 / 86.9.
constexpr int kLatentManyWaves = 8;
constexpr long long kLatentManyRows = 1 << 20;  // with more, the others' joins take longer than any one row's
struct LatentJoin {
  int waves, few;  // few: INT_MAX where every row is joined alike
};
inline LatentJoin latent_join(long long mean, long long most, long long rows, bool two_passes) {
  if (mean >= 48 && rows <= 128) return LatentJoin{16, INT_MAX};
  if (mean >= 24 && rows <= 512) return LatentJoin{8, INT_MAX};
  const bool alike = most < 48 || rows > kLatentManyRows;
  return mean >= 10 ? LatentJoin{4, alike || two_passes ? INT_MAX : 48} : LatentJoin{1, alike ? INT_MAX : 12};
}
inline int latent_join_ahead(int waves) { return waves * (waves >= 8 ? 8 : 4); }

// Query rows per tile by the rows that a sequence has on average.  Us, e4m3, 64 sequences
// of 3000: 32 heads 46.9 in tiles of 32, 56.7 of 16, 48.7 of 64; 16 heads of 600 to 8000
// 50.4 of 16, 54.6 of 32; 32 of 3000, 64 heads 39.8 of 64, 45.3 of 32; 128 heads, bf16,
// 32 of 900 to 6000 58.8 of 64 against 80.6 of 32.
inline int latent_tile_rows(int T, int B, int H) {
  const long long rows = (long long)T * H / B;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

// Whether prefixes of `keys` keys at most get a pass of their own: where the steps that it saves
// pay for the partials of every row: for 2.5 steps per CU at the least, and for a step per 2560 rows and
// CU where those are more.  A step takes 1 for a tile of 16 rows, 1.7 of 32, 3 of 64; a
// sequence is one tile where it fills none of 64, a prefix's tokens are tiles of 64.  Saved steps
// and us, two passes / one: 16 heads, 64 sequences behind 8192 keys, e4m3, 2048: 49 / 69; 8 prompts of
// 2600 with 8 samples each 656: 35.4 / 36.9, 16 prompts with 4 each 656: 37.2 / 37.0; 64 behind 2000
// 512: 34.1 / 33.7; 16 behind 8192 512: 34.2 / 30.1; 21 prompts of 6000 with 3 each, bf16, none: 76 / 71; 32
// heads, 64 behind 8192 1638: 70 / 88, 32 behind 12000 1203: 66.5 / 69.2, behind 6000 602: 50.6 / 45.5.
// Many rows: 400 of 16 heads behind 1024 1600: 66 / 74; 512 of 32 heads, bf16, behind 512 819: 105 / 86, behind
// 1024 1638: 117 / 109, behind 2048 3277: 148 / 160.  Over 420 batches of 4 to 32 heads, 16 to 512 sequences and
// 1 to 64 prefixes of 400 to 9000 keys the choice takes 1% longer than the better way on average, 7% in 95 of 100;
// at most 40%: 21 prompts of 9000 with 3 sequences of 4 heads each, where the tiles of 64 are a fifth full and one
// pass is chosen.
inline bool latent_prefix_pass(int G, int B, int T, int H, long long keys) {
  const int own = latent_tile_rows(T, B, H);
  if (own == 64) return false;
  const long long tiles = plan_min(B, T), all = (long long)T * H, rows = (all + G - 1) / G;
  const long long saved = tiles * (own == 16 ? 10 : 17) - G * ((rows + 63) / 64) * 30;  // tenths, per step
  const long long least = 25LL * kLatentUnits;
  return saved > 0 && saved * ((keys + kLatentKeys - 1) / kLatentKeys) >= (all > least ? all : least);
}

}  // namespace ferret
