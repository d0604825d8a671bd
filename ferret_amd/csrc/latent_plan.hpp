// How the latent attention deals a ragged batch to its work-groups, and where a
// position's row stands in the paged cache.  Plain C++17 without HIP, so that a CPU
// test compiles it on its own and walks every work-group of many batches
// (tests/test_latent_plan.py): every (sequence, row tile, step) is taken once, no two
// pieces share a slot, the records lead to exactly the pieces of a tile, and no row
// outside the cache is named, whatever the index tensors hold.
#pragma once

#ifdef __HIPCC__
#define FERRET_HD __host__ __device__ __forceinline__
#else
#define FERRET_HD inline
#endif

namespace ferret {

constexpr int kLatentKeys = 64;    // keys per step
constexpr int kLatentUnits = 256;  // work-groups the work is dealt to: one per CU

FERRET_HD int plan_min(int a, int b) { return a < b ? a : b; }
FERRET_HD int plan_max(int a, int b) { return a > b ? a : b; }

// The row of `offset` in page `id`, -1 where id names no page.
FERRET_HD long long page_row(int id, int pages, int page_size, int offset) {
  return (unsigned)id < (unsigned)pages ? (long long)id * page_size + offset : -1;
}

// The work of one sequence: query rows (token-major, then heads) in tiles of `mr`,
// keys in steps.  Index values outside the tensors are cut to them.
struct LatentSeq {
  int q0, n, len, rows, tiles, steps;
  FERRET_HD int work() const { return tiles * steps; }
};

FERRET_HD LatentSeq latent_seq(int start, int end, int len, int T, int H, int mr, int most_keys) {
  LatentSeq s;
  s.q0 = plan_min(plan_max(start, 0), T);
  s.n = plan_min(plan_max(end, s.q0), T) - s.q0;
  s.len = plan_min(plan_max(len, 0), most_keys);
  s.rows = s.n * H;
  s.tiles = (s.rows + mr - 1) / mr;
  s.steps = plan_max((s.len + kLatentKeys - 1) / kLatentKeys, 1);  // an empty sequence's rows are written too
  return s;
}

// Steps per work-group of a line of `total`.
FERRET_HD int latent_chunk(int total, int min_steps) {
  return plan_max(min_steps, (total + kLatentUnits - 1) / kLatentUnits);
}

// The slot of the partial result that work-group `block` takes up at `cur` of the
// line: its share may start and end inside a tile, so it has two.
FERRET_HD int latent_slot(int block, int cur, int chunk) { return 2 * block + (cur > block * chunk ? 1 : 0); }

// Where the pieces of a tile stand that work-group `block` begins at `cur`: the first
// in its slot `odd`, the others each in the even slot of the next work-group.
struct LatentRecord {
  int block, pieces, odd;
};
FERRET_HD LatentRecord latent_record(int block, int cur, int steps, int chunk) {
  return LatentRecord{block, (cur + steps - 1) / chunk - block + 1, cur > block * chunk ? 1 : 0};
}
FERRET_HD int latent_record_slot(const LatentRecord& r, int piece) {
  return 2 * (r.block + piece) + (piece == 0 && r.odd != 0 ? 1 : 0);
}
// More than one piece, all of them inside the workspace (a row that no sequence
// covers has no record, and whatever stands there must lead nowhere else).
FERRET_HD bool latent_record_joins(const LatentRecord& r) {
  return r.pieces >= 2 && r.pieces <= kLatentUnits && (unsigned)r.block <= (unsigned)(kLatentUnits - r.pieces);
}

}  // namespace ferret
