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
// More than one piece, all of them inside the workspace (a row that no sequence
// covers has no record, and whatever stands there must lead nowhere else).
FERRET_HD bool latent_record_joins(const LatentRecord& r, int side) {
  return r.pieces >= 2 && r.pieces <= kLatentUnits && (unsigned)r.slot0 < (unsigned)(2 * kLatentUnits) &&
         (r.slot0 | 1) + 2 * side * (r.pieces - 1) < 2 * kLatentUnits;
}

}  // namespace ferret
