// Latent attention in its absorbed form, over the paged cache (latent.hpp): every
// head of a token attends the same rows, of which the 512 latents are key and
// value at once:
//   s_ij = scale * (ql_i . c_j + qr_i . k_j)      c_j latents, k_j rotary key
//   o_i  = sum_j softmax_j(s_ij) c_j              512 latents, expanded by the caller
// Token i of a sequence of `len` keys and n new tokens sees keys j <= len - n + i
// (causal) or all of them.  A row that sees none gives zeros and lse -inf.
//
// Work.  The n * H query rows of a sequence are cut into tiles of MR, the keys into
// tiles of 64 ("steps").  All (sequence, row tile, step) triples form one line that
// is dealt to the work-groups in equal pieces, so a ragged batch loads the card
// evenly whatever its lengths; a row tile that is cut leaves fp32 partials (O, m, l)
// in the workspace, which a second kernel joins in order (deterministic).  A
// work-group finds its piece by itself from lens and cu_q: no host read, so the
// call can be captured into a graph and replayed with other lengths.
//
// Up to 32 rows per tile (latent_attention_kernel), a step: the 64 cached rows come into
// LDS by asynchronous loads, once for key and value.  S^T = K Q^T is dealt to the waves
// by queries (WQ) and keys (WK), with the keys as MFMA rows, so that a lane holds the
// scores of one query; its softmax terms go through LDS as bf16, and for O^T = V^T P^T
// every wave takes all queries and a share of the 512 columns.  So no product is done
// twice and a row is read from LDS WQ times as key and once as value; the output tile
// stays in registers.  V^T is read with the transposing LDS loads (ds_read_b64_tr):
// 16 columns by key.  64 rows (latent_attention_wide_kernel): scores and output are
// done by waves of their own, side by side.
// e4m3 rows stay e4m3 in LDS.  Keys are widened and scaled in one instruction (exact);
// values are widened unscaled, and each probability is multiplied by its key's power
// of two instead, before (16 and 32 rows: one copy of P per block of 128 columns) or
// after (64 rows) it is rounded to bf16: exact, so nothing is lost by it.
//
// What bounds it.  16 heads, one token: the cache's bytes; 64 sequences of 600 to 8000
// keys, e4m3, 49 us, 3.6 TB/s with launch and joins, of which the kernel takes 45.  64
// rows: no one unit.  32 sequences of 8192, 128 heads, bf16, 100 us: the matrix units
// are busy for 40% of the cycles, LDS for 27%, the vector units for 20%, and memory
// delivers 3.0 TB/s; the clock falls to 2.0 GHz under it.  e4m3, 92 us: the vector
// units take 39%, widening the keys twice and the values once, beside 40% of products.
//
// Numerics: S, m, l and O are fp32; P is rounded to bf16 for the MFMA (half a step,
// 2^-8 relative, random over the keys), l sums the unrounded P.  The running
// maximum moves only when a score passes it by more than 2^8: P stays <= 256 and the
// rescaling of O, 256 registers, is skipped for nearly all steps.
#include "attention.hpp"
#include "latent.hpp"

#include <initializer_list>

namespace ferret {
namespace {

constexpr int kKeys = kLatentKeys, kUnits = kLatentUnits;
constexpr int kJoinRows = 512;  // rows up to which four work-groups join a row's pieces
constexpr int kAhead = 4;      // LDS fragments read ahead
constexpr int kFence = 4;      // fragments between scheduling fences

struct Args {
  const uint16_t *ql, *qr;
  int ql_t, ql_h, qr_t, qr_h;  // strides of tokens and heads, in elements
  const uint8_t* data;
  const uint32_t* scales;
  Pages pages;
  const int32_t *lens, *cu_q;
  int B, T, H;
  float scale_log2;  // scale * log2(e)
  int causal;
  int min_steps;
  int side_by_side;  // row tiles of a sequence taken at the same time
  uint16_t* out;  // [T, H, 512]
  float* lse;     // [T, H] or null
  // The workspace: rows [T * H] (int4), then ml [2 * kUnits][MR] (m and l), then the
  // partial outputs [2 * kUnits][MR][512].  A row's record is {first slot, pieces, row
  // in tile, -}.
  uint8_t* ws;
  __host__ __device__ int4* rows() const { return reinterpret_cast<int4*>(ws); }
  __host__ __device__ float2* ml() const {
    return reinterpret_cast<float2*>(ws + (((size_t)T * H * sizeof(int4) + 255) & ~(size_t)255));
  }
  __host__ __device__ float* part(int mr) const { return reinterpret_cast<float*>(ml() + 2 * kUnits * mr); }
};

template <int MR>
__device__ __forceinline__ LatentSeq sequence(const Args& a, int b) {
  return latent_seq(a.cu_q[b], a.cu_q[b + 1], a.lens[b], a.T, a.H, MR, a.side_by_side,
                    a.pages.max_pages * a.pages.page_size);
}

template <bool F8>
struct Tile {
  static constexpr int kRowB = F8 ? kRowE4m3 : kRowBf16;
  static constexpr int kChunks = kRowB / 16;
  static constexpr int kFrags = kRowB / 64;        // 16-byte chunks per lane of a key fragment row
  static constexpr int kLoads = 8 * kChunks / 64;  // per group of 8 rows
  static constexpr int kData = kKeys * kRowB;
  static constexpr int kBytes = kData + (F8 ? kKeys * 4 : 0);  // then the scale words
  static constexpr int kBufs = F8 ? 3 : 2;
  static constexpr int vmem(int waves) { return 8 / waves * kLoads + (F8 ? 1 : 0); }  // loads of a wave per step
};

// What only the ends of a piece need, the arguments among it, kept in LDS: scalar
// registers are short.
struct Side {
  Args args;
  int chunk, extra;      // the deal
  int seq_at, b;         // the sequence at hand and its place on the line
  LatentSeq seq;
  int first_row;         // the tile's first row among all [T * H]
  int slot;              // of the partial result, -1 for a whole tile
  int end;               // of this work-group's share of the line
};

// By fields: a struct's copy would stand in scratch memory.
__device__ __forceinline__ void put_seq(LatentSeq* to, const LatentSeq& s) {
  to->q0 = s.q0;
  to->n = s.n;
  to->len = s.len;
  to->rows = s.rows;
  to->groups = s.groups;
  to->steps = s.steps;
}
__device__ __forceinline__ LatentSeq get_seq(const LatentSeq* from) {
  return LatentSeq{from->q0, from->n, from->len, from->rows, from->groups, from->steps};
}

__device__ __forceinline__ void put_args(Args* to, const Args& a) {
  to->ql = a.ql;
  to->qr = a.qr;
  to->ql_t = a.ql_t;
  to->ql_h = a.ql_h;
  to->qr_t = a.qr_t;
  to->qr_h = a.qr_h;
  to->pages.table = a.pages.table;
  to->pages.max_pages = a.pages.max_pages;
  to->pages.pages = a.pages.pages;
  to->pages.page_size = a.pages.page_size;
  to->lens = a.lens;
  to->cu_q = a.cu_q;
  to->B = a.B;
  to->T = a.T;
  to->H = a.H;
  to->causal = a.causal;
  to->side_by_side = a.side_by_side;
  to->out = a.out;
  to->lse = a.lse;
  to->ws = a.ws;
}

// LDS after the tile buffers.
template <int MR, int WK, bool F8>
struct Lds {
  static constexpr int kCopies = F8 ? 4 : 1;
  static constexpr int kP = Tile<F8>::kBufs * Tile<F8>::kBytes;  // P [copy][query][64 keys] bf16
  static constexpr int kTop = kP + kCopies * MR * 128;           // maxima [WK][MR], then factors [MR]
  static constexpr int kValid = kTop + (WK + 1) * MR * 4;        // validity of the 16-row blocks, per buffer
  static constexpr int kMove = kValid + 16;                      // which waves saw the maximum move
  static constexpr int kSide = kMove + 16;
  static constexpr int kBytes = kSide + sizeof(Side);
};
static_assert(Lds<32, 4, true>::kBytes <= 160 * 1024 && Lds<32, 4, false>::kBytes <= 160 * 1024, "LDS of a CU");

// Chunk c (16 bytes) of row r stands at chunk c ^ swz(r): the rows of two transposed
// blocks (4 rows of two chunks each, or 8 of one) fall on distinct banks (a row is 32
// banks past a multiple of 64), and so do the 16 lanes of a key fragment that are read
// together, which are not neighbours: rows 0 - 3 and 12 - 15 of one chunk with 4 - 11 of
// the next.  Bit 2 without r & 4, which suits 16 neighbours only, had four times the
// bank conflicts (38% of the LDS cycles of 128 heads, bf16) and 2% more time.
__device__ __forceinline__ int swz(int r) { return (((r >> 1) ^ r) & 4) | (r & 2) | ((r >> 2) & 1); }

// The start of a work-group's share of the line: false where it has none.  The page
// table's first lines come under the loads of the lengths.  tot: 24 words of LDS.
template <int MR, int NT>
__device__ __forceinline__ bool take_share(const Args& a, LatentPlace place, Side* side, int* tot, int* cur) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int near =
      a.pages.table[(long long)latent_near(place.unit, kUnits / a.side_by_side, a.B) * a.pages.max_pages];
  const int per = (a.B + NT - 1) / NT;
  const int b0 = threadIdx.x * per;
  LatentSeq s{};
  int mine = 0, my_groups = 0;
  for (int i = 0; i < per && b0 + i < a.B; ++i) {
    s = sequence<MR>(a, b0 + i);
    mine = latent_add(mine, s.work(0));
    my_groups = latent_add(my_groups, s.groups);
  }
  int incl = mine, incl_groups = my_groups;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, 64), og = __shfl_up(incl_groups, off, 64);
    if (lane >= off) {
      incl = latent_add(incl, o);
      incl_groups = latent_add(incl_groups, og);
    }
  }
  constexpr int NW = NT / 64;
  if (lane == 63) {
    tot[wave] = incl;
    tot[NW + wave] = incl_groups;
  }
  __syncthreads();
  asm volatile("" ::"v"(near));
  int before = 0, all = 0, groups_before = 0, groups = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) {
      before = latent_add(before, tot[w]);
      groups_before = latent_add(groups_before, tot[NW + w]);
    }
    all = latent_add(all, tot[w]);
    groups = latent_add(groups, tot[NW + w]);
  }
  const int units = kUnits / a.side_by_side;
  bool whole = false;
  if (per == 1) {  // more sequences than threads do not all fit
    const bool fits = latent_fits(s, latent_chunk(all, units, a.min_steps));
    if (lane == 0) tot[2 * NW + wave] = 0;
    if (__any(!fits) && lane == 0) tot[2 * NW + wave] = 1;
    __syncthreads();
    int misfits = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) misfits |= tot[2 * NW + w];
    whole = misfits == 0;
  }
  const LatentDeal deal = latent_deal(all, groups, whole, units, a.min_steps);
  const int total = deal.total, chunk = deal.chunk, extra = deal.extra;
  const int start = (int)min((long long)place.unit * chunk, (long long)total);
  if (start >= total) return false;
  const int excl = before + incl - mine + extra * (groups_before + incl_groups - my_groups);
  if (excl <= start && start < excl + mine + extra * my_groups) {
    int at = excl, i = 0;
    if (per > 1)
      for (;; ++i) {
        s = sequence<MR>(a, b0 + i);
        if (start < at + s.work(extra) || i + 1 == per) break;
        at += s.work(extra);
      }
    side->b = b0 + i;
    put_seq(&side->seq, s);
    side->seq_at = at;
    side->chunk = chunk;
    side->extra = extra;
    side->end = min(start + chunk, total);
    put_args(&side->args, a);
  }
  *cur = uniform(start);
  __syncthreads();
  return true;
}

// A piece of a row tile: steps s0 .. s1 of sequence b.
struct Piece {
  int b, s0, s1, len, past, q0;
  bool one;               // the sequence has one new token
  int row0, row_last;     // query rows of the sequence
  int see_all, see_any;   // keys that the first and the last token of the tile see
};

// The piece at `cur`, its place noted in LDS and its rows' record in the workspace;
// false where there are no keys (the extra steps) or no rows (fewer tiles than
// work-groups side by side).
template <int MR>
__device__ __forceinline__ bool next_piece(LatentPlace place, Side* side, int cur, Piece* p) {
  const Args& in = side->args;
  const int extra = side->extra;
  int b = uniform(side->b), seq_at = uniform(side->seq_at);
  LatentSeq s = get_seq(&side->seq);
  while (cur >= seq_at + s.work(extra) && b + 1 < in.B) {  // the next sequence with rows
    seq_at += s.work(extra);
    s = sequence<MR>(in, ++b);
  }
  p->b = b = uniform(b);
  p->len = uniform(s.len);
  p->q0 = uniform(s.q0);
  const int steps = uniform(s.steps), line = uniform(s.steps + extra), n = uniform(s.n);
  const int group = s.groups > 1 ? uniform((cur - seq_at) / line) : 0;
  p->s0 = uniform(cur - seq_at - group * line);
  p->s1 = uniform(min(line, p->s0 + (side->end - cur)));
  p->row0 = uniform((group * in.side_by_side + place.lane) * MR);
  p->row_last = uniform(min(p->row0 + MR, s.rows) - 1);
  if (p->row_last < p->row0 || p->s0 >= steps) return false;
  p->past = p->len - n + 1;
  const bool causal = in.causal && n > 1;  // one token sees all
  p->see_all = causal ? uniform(max(p->past + p->row0 / in.H, 0)) : p->len;
  p->see_any = causal ? uniform(max(p->past + p->row_last / in.H, 0)) : p->len;
  p->one = n == 1;
  const int chunk = side->chunk, first_row = p->q0 * in.H + p->row0;
  __syncthreads();  // the piece before is done with its record and buffers
  if (threadIdx.x == 0) {
    side->b = b;
    put_seq(&side->seq, s);
    side->seq_at = seq_at;
    side->first_row = first_row;
    side->slot =
        p->s0 == 0 && p->s1 >= steps ? -1 : latent_slot(place.unit, place.lane, in.side_by_side, cur, chunk);
  }
  if (p->s0 == 0 && (int)threadIdx.x <= p->row_last - p->row0) {
    const LatentRecord r = latent_record(place.unit, place.lane, in.side_by_side, cur, steps, chunk);
    in.rows()[first_row + threadIdx.x] = make_int4(r.slot0, r.pieces, threadIdx.x, 0);
  }
  return true;
}

// Where 16-row block `block` (of the sequence) of the wave's lanes stands in the cache, in
// units of 16 rows, -1 where it has no page.
__device__ __forceinline__ int find_block(const Pages& pages, const int32_t* table, int block) {
  const int pos = block * 16, page = pos / pages.page_size;
  const int id = pos >= 0 && page < pages.max_pages ? table[page] : -1;
  const long long row = page_row(id, pages.pages, pages.page_size, pos - page * pages.page_size);
  return row < 0 ? -1 : (int)(row >> 4);
}

// A fragment of queries (column r16 = row `r` of the sequence), and the keys that it sees.
template <bool F8>
__device__ __forceinline__ int get_queries(const Args& in, const Piece& p, int r, int g, u32x4 (&qf)[18]) {
  const int rc = min(r, p.row_last), tok = p.one ? 0 : rc / in.H, head = rc - tok * in.H;  // past the tile: its last row
  const uint16_t* ql = in.ql + (long long)(p.q0 + tok) * in.ql_t + (long long)head * in.ql_h;
  const uint16_t* qr = in.qr + (long long)(p.q0 + tok) * in.qr_t + (long long)head * in.qr_h;
#pragma unroll
  for (int k = 0; k < 16; ++k) qf[k] = ld_u32x4(ql + (F8 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g));
#pragma unroll
  for (int k = 0; k < 2; ++k) qf[16 + k] = ld_u32x4(qr + 32 * k + 8 * g);
  return r <= p.row_last ? max(in.causal ? p.past + tok : p.len, 0) : 0;
}

// Inf and NaN among 16 bytes of values become zeros.
template <bool F8>
__device__ __forceinline__ u32x4 only_finite(u32x4 v) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (F8) {
      const uint32_t nan = (((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
      v[w] &= ~(nan * 255u);
    } else {
      if ((v[w] & 0x7f80u) == 0x7f80u) v[w] &= 0xffff0000u;
      if ((v[w] & 0x7f800000u) == 0x7f800000u) v[w] &= 0x0000ffffu;
    }
  }
  return v;
}

// A value that a row does not see must not reach it as 0 * NaN: before the products with a
// step's values, rows of the step (the first of which is key `first`) that no query of the
// tile sees become zeros, and Inf and NaN of rows that some do not see are cleared.  Each
// wave does so for its own columns, CT blocks of 16 from chunk `chunk` on.  ok: which 16-row
// blocks have a page.
// A query that sees a cleared Inf or NaN has NaN in its l, as its key is the same row; but
// a key of bf16 latents with an Inf may score -inf and have no weight, and 0 * Inf makes
// that column NaN in the steps that all queries see: so it does here.
template <bool F8, int STEP, int CT, int WQ>
__device__ __forceinline__ void clear_unseen(const Args& in, const Piece& p, uint8_t* buf, int first, uint32_t ok,
                                             int chunk, f32x4 (&o)[CT][WQ]) {
  constexpr int VC = F8 ? CT : 2 * CT, ROW = F8 ? kRowE4m3 : kRowBf16;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const auto place = [&](int r, int c) { return buf + r * ROW + (((chunk + c) ^ swz(r)) << 4); };
  // Every row seen by all or by none: a loop of its own where scalar registers are left for it
  // (128 heads, bf16, 32 sequences of 900 to 6000: 58.5 us, 59.3 without).
  if (WQ == 4 && p.see_all >= p.see_any) {
#pragma unroll 1
    for (int i0 = 0; i0 < STEP * VC; i0 += 64) {
      const int r = (i0 + lane) / VC;
      if (first + r >= p.see_any || !((ok >> (8 * (r >> 4))) & 1))
        *reinterpret_cast<u32x4*>(place(r, lane % VC)) = u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
#pragma unroll 1
  for (int i0 = 0; i0 < STEP * VC; i0 += 64) {
    const int r = (i0 + lane) / VC, key = first + r;
    const bool none = key >= p.see_any || !((ok >> (8 * (r >> 4))) & 1), some = !none && key >= p.see_all;
    u32x4* const at = reinterpret_cast<u32x4*>(place(r, lane % VC));
    u32x4 x = {0u, 0u, 0u, 0u}, fine = x;
    if (some) fine = only_finite<F8>(x = *at);
    if (!F8 && p.see_all < p.see_any) {
      const bool bad = x[0] != fine[0] || x[1] != fine[1] || x[2] != fine[2] || x[3] != fine[3];
      for (unsigned long long rest = __ballot(bad); rest != 0;) {
        const int first_bad = __ffsll((long long)rest) - 1, row = (i0 + first_bad) / VC;
        rest &= ~0ull << (first_bad / VC * VC + VC - 1) << 1;  // the row's other chunks are looked at with it
        uint32_t sees[WQ];  // all bits where the lane's query sees the key
#pragma unroll
        for (int f = 0; f < WQ; ++f) {
          const int tok = p.one ? 0 : min(p.row0 + f * 16 + r16, p.row_last) / in.H;
          sees[f] = first + row < (in.causal ? p.past + tok : p.len) ? ~0u : 0u;
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) {  // the lane's columns c * 16 + 4g .. 4g + 3
          const u32x2 w = *reinterpret_cast<const u32x2*>(place(row, 2 * c + (g >> 1)) + (g & 1) * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t inf = j & 1 ? 0x7f800000u : 0x7f80u;
            const uint32_t nan = (w[j >> 1] & inf) == inf ? 0x7fc00000u : 0u;
#pragma unroll
            for (int f = 0; f < WQ; ++f) {
              const float v = o[c][f][j];  // copied first: a bit cast of a vector's element reads element 0
              o[c][f][j] = __uint_as_float(__float_as_uint(v) | (nan & sees[f]));
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      asm volatile("" ::: "memory");
    }
    if (none || some) *at = fine;
  }
}

// Row r of the tile done: its output, or its part of a piece.  o: blocks of 16 columns
// from `col` on, 4 of each per lane.
template <int MR, int CT, int WQ>
__device__ __forceinline__ void put_rows(const Side* side, const Piece& p, int f, int r16, int col,
                                         bool stats, float top, float sum, const f32x4 (&o)[CT][WQ]) {
  const Args& in = side->args;
  const int r = f * 16 + r16, slot = uniform(side->slot);
  if (p.row0 + r > p.row_last) return;
  if (slot < 0) {
    const long long at = side->first_row + r;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* to = in.out + at * kLatent + col;
#pragma unroll
    for (int c = 0; c < CT; ++c)
      *reinterpret_cast<u32x2*>(to + c * 16) =
          u32x2{pack_bf16x2(o[c][f][0] * inv, o[c][f][1] * inv), pack_bf16x2(o[c][f][2] * inv, o[c][f][3] * inv)};
    if (stats && in.lse != nullptr)
      in.lse[at] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  } else {
    const long long at = (long long)slot * MR + r;
    if (stats) in.ml()[at] = make_float2(top, sum);
    float* to = in.part(MR) + at * kLatent + col;
#pragma unroll
    for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4*>(to + c * 16) = o[c][f];
  }
}

// WQ x WK waves: 16 queries x 64 / WK keys each for the scores, all queries x
// 512 / (WQ WK) columns for the output.
template <int WQ, int WK, bool F8>
__global__ __launch_bounds__(64 * WQ * WK, WQ * WK / 4) void latent_attention_kernel(Args a) {
  using L = Tile<F8>;
  constexpr int MR = 16 * WQ, NW = WQ * WK, NT = 64 * NW;
  using M = Lds<MR, WK, F8>;
  constexpr int KT = kKeys / 16 / WK;     // 16-key blocks of a wave's scores
  constexpr int CT = kLatent / 16 / NW;   // 16-column blocks of a wave's output
  constexpr int RG = 8 / NW;              // groups of 8 rows that a wave loads
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int wq = wave / WK, wk = wave % WK;
  float* const tops = reinterpret_cast<float*>(lds + M::kTop);
  Side* const side = reinterpret_cast<Side*>(lds + M::kSide);

  const LatentPlace place = latent_place(blockIdx.x, a.side_by_side);
  int cur;
  if (!take_share<MR, NT>(a, place, side, reinterpret_cast<int*>(lds), &cur)) return;
  const Args& in = side->args;
  const uint8_t* const data = a.data;
  const uint32_t* const scales = a.scales;
  const float scale_log2 = a.scale_log2;

  // ---- lane constants
  int load_off[L::kLoads];  // source bytes within a group of 8 rows; the swizzle differs in odd groups
#pragma unroll
  for (int j = 0; j < L::kLoads; ++j) {
    const int slot = j * 64 + lane, row = slot / L::kChunks, pos = slot % L::kChunks;
    load_off[j] = row * L::kRowB + ((pos ^ swz(RG == 1 ? (wave & 1) * 8 + row : row)) << 4);
  }

  while (cur < uniform(side->end)) {
    Piece pc;
    const bool there = next_piece<MR>(place, side, cur, &pc);
    const int s0 = pc.s0, see_all = pc.see_all, see_any = pc.see_any;
    cur += pc.s1 - s0;
    if (!there) continue;
    const int last = min(pc.s1, (see_any + kKeys - 1) / kKeys);

    f32x4 o[CT][WQ];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int f = 0; f < WQ; ++f)
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][f] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The page table, 64 steps at a time: lane i holds where the 16 rows stand that the
    // wave loads from (RG groups of 8 of them) in step held + i.
    const int32_t* table = in.pages.table + (long long)pc.b * in.pages.max_pages;
    int held = s0, where;
    const auto look_up = [&]() __attribute__((always_inline)) {
      where = find_block(in.pages, table, min(held + lane, last - 1) * (kKeys / 16) + wave * RG / 2);
    };
    look_up();

    // Step t's rows into its buffer, load by load.
    const uint8_t* src;
    const uint32_t* src_scales;
    uint32_t dst, dst_scales;
    const auto aim = [&](int t) __attribute__((always_inline)) {
      if (t == held + 64) {
        held = t;
        look_up();
      }
      const int at = __builtin_amdgcn_readlane(where, t - held);
      const bool ok = at >= 0;
      const long long row = (ok ? (long long)at << 4 : 0) + (RG == 1 ? (wave & 1) * 8 : 0);  // no page: some row, masked
      if (lane == 0) lds[M::kValid + (t % L::kBufs) * 4 + wave * RG / 2] = ok ? 1 : 0;
      src = data + row * L::kRowB;
      dst = uniform(lds_address(lds) + (t % L::kBufs) * L::kBytes + wave * RG * 8 * L::kRowB);
      if constexpr (F8) {
        src_scales = scales + row;
        dst_scales = uniform(lds_address(lds) + (t % L::kBufs) * L::kBytes + L::kData + wave * RG * 32);
      }
    };
    constexpr int LD = L::vmem(NW);
    const auto load = [&](int i) __attribute__((always_inline)) {
      if (F8 && i == LD - 1) {
        if (lane < RG * 8) dma_4(src_scales, lane * 4, dst_scales);
      } else if (i < L::kLoads) {
        dma_16(src, load_off[i], dst + i * 1024);
      } else {  // the odd group: one bit of the swizzle differs
        dma_16(src + 8 * L::kRowB, load_off[i - L::kLoads] ^ 64, dst + 8 * L::kRowB + (i - L::kLoads) * 1024);
      }
    };

    u32x4 qf[18];  // queries: B fragments
    const int sees = get_queries<F8>(in, pc, pc.row0 + wq * 16 + r16, g, qf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < L::kBufs - 1; ++i)
      if (s0 + i < last) {
        aim(s0 + i);
#pragma unroll
        for (int j = 0; j < LD; ++j) load(j);
      }
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<0>();  // the queries, so that no wait for them stands in the loop; the first steps come with them
    __builtin_amdgcn_sched_barrier(0);

    for (int t = s0; t < last; ++t) {
      // Step t has landed for every wave, and the buffer refilled below has been read.
      if (L::kBufs == 3 && t + 1 < last) wait_vmcnt<LD>();
      else wait_vmcnt<0>();
      lds_barrier();
      const bool more = t + L::kBufs - 1 < last;
      if (more) aim(t + L::kBufs - 1);
      __builtin_amdgcn_sched_barrier(0);
      uint8_t* buf = lds + (t % L::kBufs) * L::kBytes;
      const uint32_t* words = reinterpret_cast<const uint32_t*>(buf + L::kData);

      // ---- S^T: 16 keys x 16 queries per block.  Key fragments are read kAhead
      // fragments before their use; the scheduling fences keep the compiler from
      // hoisting more of them than the registers hold.  The next step's loads are
      // issued in between: in one go they would hold the wave up for as long as the
      // products take.
      constexpr int CH = KT == 1 ? 2 : 1;  // chains of accumulation per block
      f32x4 sc[KT * CH];
#pragma unroll
      for (int k = 0; k < KT * CH; ++k) sc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      {
        // chunk 4j + g: the swizzle touches 8 chunks at most, j >> 1 is an offset
        const uint8_t* row = buf + (wk * KT * 16 + r16) * L::kRowB;
        const uint8_t* const at[2] = {row + ((g ^ swz(r16)) << 4), row + (((4 + g) ^ swz(r16)) << 4)};
        uint32_t word[KT];
        if constexpr (F8)
#pragma unroll
          for (int k = 0; k < KT; ++k) word[k] = words[(wk * KT + k) * 16 + r16];
        constexpr int NF = KT * L::kFrags;
        const auto frag = [&](int i) {  // i = (chunk, block)
          const int j = i / KT, k = i % KT;
          return ld_u32x4(at[j & 1] + k * 16 * L::kRowB + (j >> 1) * 128);
        };
        u32x4 ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = frag(i);
        static_for<0, NF>([&](auto ic) {
          constexpr int i = decltype(ic)::value, j = i / KT, k = i % KT;
          const u32x4 c = ring[i % kAhead];
          if constexpr (i + kAhead < NF) ring[i % kAhead] = frag(i + kAhead);
          if constexpr (F8 && j < 8) {
            const float e = __uint_as_float(((word[k] >> (8 * (j >> 1))) & 255u) << 23);
            const bf16x8 lo = e4m3x8_to_bf16x8_scaled(c[0], c[1], e), hi = e4m3x8_to_bf16x8_scaled(c[2], c[3], e);
            sc[k] = mfma_bf16(lo, __builtin_bit_cast(bf16x8, qf[2 * j]), sc[k]);
            sc[k + (CH - 1)] = mfma_bf16(hi, __builtin_bit_cast(bf16x8, qf[2 * j + 1]), sc[k + (CH - 1)]);
          } else {
            constexpr int at = CH == 2 ? j & 1 : k;
            sc[at] = mfma_bf16_16x16x32(c, qf[F8 ? j + 8 : j], sc[at]);
          }
          if constexpr (i % kFence == kFence - 1) {
            constexpr int x0 = (i + 1 - kFence) * LD / NF, x1 = (i + 1) * LD / NF;
            if (more) static_for<x0, x1>([&](auto x) { load(decltype(x)::value); });
            __builtin_amdgcn_sched_barrier(0);
          }
        });
        constexpr int rest = NF / kFence * kFence * LD / NF;
        if (more) static_for<rest, LD>([&](auto x) { load(decltype(x)::value); });
        if constexpr (CH == 2) sc[0] += sc[1];
      }
      __builtin_amdgcn_sched_barrier(0);

      // ---- masks: only where the step passes what some row sees, or misses a page
      const uint32_t ok = uniform(*reinterpret_cast<const uint32_t*>(lds + M::kValid + (t % L::kBufs) * 4));
      if ((t + 1) * kKeys > see_all || ok != 0x01010101u) {
        const int left = sees - (t * kKeys + wk * KT * 16 + 4 * g);
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int upto = (ok >> (8 * (wk * KT + k))) & 1 ? left - k * 16 : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[k][i] = i < upto ? sc[k][i] : -INFINITY;
        }
        lds_barrier();  // the keys have been read
        clear_unseen<F8, kKeys>(in, pc, buf, t * kKeys, ok, wave * CT * (F8 ? 1 : 2), o);
        if constexpr (F8) {
          if (threadIdx.x < kKeys) {
            const int r = threadIdx.x;
            if (t * kKeys + r >= see_any || !((ok >> (8 * (r >> 4))) & 1))
              reinterpret_cast<uint32_t*>(buf + L::kData)[r] = 0x7f7f7f7fu;
          }
          lds_barrier();  // the scale words are read next
        }
      }

      // ---- softmax terms of the lane's query (column r16), with the maximum of the
      // steps before
      float top = sc[0][0];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[k][i]);
      top = rows_max(top) * scale_log2;
      const bool move = __any(top > m + kLazy);  // from -inf: any finite score
      const int q = wq * 16 + r16;
      if (g == 0) tops[wk * MR + q] = top;
      if (lane == 0) lds[M::kMove + wave] = move ? 1 : 0;
      float pend;  // this step's part of l
      const auto put_p = [&]() __attribute__((always_inline)) {
        const float base = m == -INFINITY ? 0.f : m;
        pend = 0.f;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          f32x4 p;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(sc[k][i], scale_log2, -base));
            pend += p[i];
          }
          const int kb = wk * KT + k;  // 16-key block of the step: 2 chunks
          uint8_t* to = lds + M::kP + q * 128 + (((2 * kb + (g >> 1)) ^ (r16 >> 1)) << 4) + (g & 1) * 8;
          if constexpr (F8) {
            const u32x4 w4 = *reinterpret_cast<const u32x4*>(words + kb * 16 + 4 * g);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float e[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) e[i] = p[i] * __uint_as_float(((w4[i] >> (8 * c)) & 255u) << 23);
              *reinterpret_cast<u32x2*>(to + c * MR * 128) = u32x2{pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3])};
            }
          } else {
            *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])};
          }
        }
      };
      put_p();
      lds_barrier();
      const u32x2 moves = *reinterpret_cast<const u32x2*>(lds + M::kMove);

      // ---- O^T += V^T P^T, 32 keys at a time: lane (column r16, key octet g)
      const uint8_t* pbuf = lds + M::kP + (F8 ? wave * CT / 8 * MR * 128 : 0) + r16 * 128;
      const uint8_t* const pat[2] = {pbuf + ((g ^ (r16 >> 1)) << 4), pbuf + (((4 + g) ^ (r16 >> 1)) << 4)};
      u32x4 p[WQ];
      const auto get_p = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < WQ; ++f) p[f] = ld_u32x4(pat[h] + f * 16 * 128);
      };
      get_p(0);
      if (uniform(NW == 8 ? moves[0] | moves[1] : moves[0]) != 0) {
        // The maximum of some query moves: again with the new one, O follows.
        float to = m;
#pragma unroll
        for (int w = 0; w < WK; ++w) to = fmaxf(to, tops[w * MR + q]);
        const float by = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= by;
        if (wk == 0 && g == 0) tops[WK * MR + q] = by;
        lds_barrier();  // P has been read
        put_p();
        lds_barrier();
        get_p(0);
#pragma unroll
        for (int f = 0; f < WQ; ++f) {
          const float by = tops[WK * MR + f * 16 + r16];
#pragma unroll
          for (int c = 0; c < CT; ++c) o[c][f] *= by;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      l += pend;
      __builtin_amdgcn_sched_barrier(0);
      {
        // An exclusive-or of the block into the address is the swizzle: a wave's columns
        // start on a multiple of its chunks, and the bits below belong to the swizzle.
        constexpr int WB = CT * (F8 ? 16 : 32);  // a wave's bytes of a row
        const int row = 8 * g + (F8 ? r16 >> 1 : r16 >> 2);
        const int z = ((swz(row) ^ (F8 ? 0 : (lane >> 1) & 1)) << 4) ^ (wave * WB & 127);
        const uint32_t at = (uint32_t)(t % L::kBufs) * L::kBytes + row * L::kRowB + (wave * WB & ~127) + z + 8 * (lane & 1);
        const auto frag = [&](int i) {  // i = (half, block)
          const int h = i / CT, c = i % CT;
          if constexpr (F8) {
            const u32x2 v = lds_tr8(lds + (at ^ (c << 4)) + h * 32 * L::kRowB);
            return u32x4{v[0], v[1], 0u, 0u};
          } else {  // rows 4 further: bits 0 and 2 of the swizzle flip
            const uint8_t* x = lds + (at ^ ((c & 3) << 5)) + (c >> 2) * 128 + h * 32 * L::kRowB;
            const uint8_t* x4 = lds + (at ^ ((c & 3) << 5) ^ 80) + (c >> 2) * 128 + (h * 32 + 4) * L::kRowB;
            const u32x2 v0 = lds_tr16(x), v1 = lds_tr16(x4);
            return u32x4{v0[0], v0[1], v1[0], v1[1]};
          }
        };
        u32x4 ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = frag(i);
        static_for<0, kKeys / 32>([&](auto hc) {
          constexpr int h = decltype(hc)::value;
          if constexpr (h > 0) get_p(h);
          static_for<0, CT>([&](auto cc) {
            constexpr int c = decltype(cc)::value, i = h * CT + c;
            const u32x4 v = ring[i % kAhead];
            if constexpr (i + kAhead < kKeys / 32 * CT) ring[i % kAhead] = frag(i + kAhead);
            const bf16x8 vb = F8 ? e4m3x8_to_bf16x8(v[0], v[1]) : __builtin_bit_cast(bf16x8, v);
#pragma unroll
            for (int f = 0; f < WQ; ++f) o[c][f] = mfma_bf16(vb, __builtin_bit_cast(bf16x8, p[f]), o[c][f]);
            if constexpr (i % kFence == kFence - 1) __builtin_amdgcn_sched_barrier(0);
          });
        });
      }
    }

    // ---- the piece's result: l of all waves, then each wave's columns
    __syncthreads();  // the last step's maxima and factors have been read
    {
      float sum = l;
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      const int q = wq * 16 + r16;
      if (g == 0) tops[wk * MR + q] = sum;
      if (wk == 0 && g == 0) tops[WK * MR + q] = m;
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < WQ; ++f) {
      float sum = tops[f * 16 + r16];
#pragma unroll
      for (int w = 1; w < WK; ++w) sum += tops[w * MR + f * 16 + r16];
      put_rows<MR>(side, pc, f, r16, wave * CT * 16 + 4 * g, wave == 0 && g == 0, tops[WK * MR + f * 16 + r16],
                   sum, o);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// ---- 64 query rows: two products at a time

// A step is 32 keys (bf16) or 64 (e4m3).  LDS: the buffers (one step's values, one's
// keys, the others on their way), P twice, and the small records.
template <bool F8>
struct Wide {
  static constexpr int kRows = 64, kStep = F8 ? 64 : 32, kBufs = F8 ? 3 : 4, kAway = kBufs - 2;
  static constexpr int kData = kStep * Tile<F8>::kRowB, kBytes = kData + (F8 ? kStep * 4 : 0);
  static constexpr int kPRow = kStep * 2, kPBytes = kRows * kPRow;
  static constexpr int kP = kBufs * kBytes;             // P [2][query][keys] bf16
  static constexpr int kTop = kP + 2 * kPBytes;         // maxima [2][64], factors [64]
  static constexpr int kFin = kTop + 3 * kRows * 4;     // sums [2][64], maxima [64] of the piece
  static constexpr int kFlags = kFin + 3 * kRows * 4;   // per step parity: which waves saw the maximum move [4],
  static constexpr int kValid = kFlags + 16;            // per buffer: validity of its 16-row blocks [4]
  static constexpr int kSide = kValid + 16;
  static constexpr int kLds = kSide + sizeof(Side);
  static constexpr int kGroups = kStep / 32;                                  // groups of 8 rows that a wave loads
  static constexpr int kLoad = kGroups * Tile<F8>::kLoads + (F8 ? 1 : 0);     // its loads per step
};
static_assert(Wide<true>::kLds <= 160 * 1024 && Wide<false>::kLds <= 160 * 1024, "LDS of a CU");

// Waves 0 - 3 take the scores of one step (32 queries and half of the keys each) while
// waves 4 - 7, one of them on every SIMD beside one of the others, add the step before
// to the output (64 queries x 128 columns each) and load the keys to come: the matrix
// unit is fed by one while the other is at its softmax, at a barrier or at its loads,
// and neither holds more than half of the registers (Q is 144, O 128 of 256).
template <bool F8>
__global__ __launch_bounds__(512, 2) void latent_attention_wide_kernel(Args a) {
  using L = Tile<F8>;
  using M = Wide<F8>;
  constexpr int MR = M::kRows, KT = M::kStep / 32;  // 16-key blocks of a wave's scores
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  float* const tops = reinterpret_cast<float*>(lds + M::kTop);
  float* const fin = reinterpret_cast<float*>(lds + M::kFin);
  Side* const side = reinterpret_cast<Side*>(lds + M::kSide);
  // P of a query: chunk c of 8 keys stands at c ^ swz_p(query)
  const int zp = M::kStep == 64 ? r16 >> 1 : r16 >> 2;

  const LatentPlace place = latent_place(blockIdx.x, a.side_by_side);
  int cur;
  if (!take_share<MR, 512>(a, place, side, reinterpret_cast<int*>(lds), &cur)) return;
  const Args& in = side->args;
  const float scale_log2 = a.scale_log2;

  if (wave < 4) {
    // ================ scores
    const int wq = wave >> 1, wk = wave & 1;
    while (cur < uniform(side->end)) {
      Piece pc;
      const bool there = next_piece<MR>(place, side, cur, &pc);
      cur += pc.s1 - pc.s0;
      if (!there) continue;
      const int u0 = pc.s0 * (64 / M::kStep);
      const int end = min(pc.s1 * (64 / M::kStep), (pc.see_any + M::kStep - 1) / M::kStep);
      u32x4 qf[2][18];
      int sees[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) sees[f] = get_queries<F8>(in, pc, pc.row0 + (wq * 2 + f) * 16 + r16, g, qf[f]);
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, pend[2] = {0.f, 0.f};
      f32x4 sc[KT][2];

      // P of step u from its scores and the maxima so far
      const auto put_p = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const float base = m[f] == -INFINITY ? 0.f : m[f];
          pend[f] = 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            f32x4 p;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              p[i] = __builtin_amdgcn_exp2f(fmaf(sc[k][f][i], scale_log2, -base));
              pend[f] += p[i];
            }
            const int q = (wq * 2 + f) * 16 + r16, chunk = 2 * (wk * KT + k) + (g >> 1);
            *reinterpret_cast<u32x2*>(lds + M::kP + (u & 1) * M::kPBytes + q * M::kPRow + ((chunk ^ zp) << 4) + (g & 1) * 8) =
                u32x2{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])};
          }
        }
      };

      for (int u = u0; u <= end && end > u0; ++u) {
        lds_barrier();  // step u has landed, P of the step before is there
        // Everything that the step reads first goes out before anything is waited for.
        const int buffer = u % M::kBufs;
        const int flags = *reinterpret_cast<const int*>(lds + M::kFlags + ((u & 1) ^ 1) * 4);
        const uint32_t valid = *reinterpret_cast<const uint32_t*>(lds + M::kValid + buffer * 4);
        const uint8_t* buf = lds + buffer * M::kBytes;
        const uint8_t* row = buf + (wk * KT * 16 + r16) * L::kRowB;
        const uint8_t* const at[2] = {row + ((g ^ swz(r16)) << 4), row + (((4 + g) ^ swz(r16)) << 4)};
        uint32_t word[KT];
        if constexpr (F8)
#pragma unroll
          for (int k = 0; k < KT; ++k)
            word[k] = reinterpret_cast<const uint32_t*>(buf + M::kData)[(wk * KT + k) * 16 + r16];
        constexpr int NF = KT * L::kFrags;
        const auto frag = [&](int i) {  // i = (chunk, block)
          const int j = i / KT, k = i % KT;
          return ld_u32x4(at[j & 1] + k * 16 * L::kRowB + (j >> 1) * 128);
        };
        u32x4 ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = frag(i);
        if (u > u0) {
          if (uniform(flags) != 0) {  // the maximum of some query moves: again with the new one, O follows
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const int q = (wq * 2 + f) * 16 + r16;
              const float to = fmaxf(m[f], fmaxf(tops[q], tops[MR + q]));
              const float by = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[f] - to);
              m[f] = to;
              l[f] *= by;
              if (wk == 0 && g == 0) tops[2 * MR + q] = by;
            }
            put_p(u - 1);
            lds_barrier();
          }
          l[0] += pend[0];
          l[1] += pend[1];
        }
        if (u == end) break;
        __builtin_amdgcn_sched_barrier(0);

        // ---- S^T: key fragments read kAhead before their use, four chains of accumulation
        f32x4 part[2][2];
#pragma unroll
        for (int f = 0; f < 2; ++f) part[f][0] = part[f][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        static_for<0, NF>([&](auto ic) {
          constexpr int i = decltype(ic)::value, j = i / KT, k = i % KT;
          const u32x4 c = ring[i % kAhead];
          if constexpr (i + kAhead < NF) ring[i % kAhead] = frag(i + kAhead);
          if constexpr (F8 && j < 8) {
            constexpr int lo_at = KT == 2 ? k : 0, hi_at = KT == 2 ? k : 1;
            const float e = __uint_as_float(((word[k] >> (8 * (j >> 1))) & 255u) << 23);
            const bf16x8 lo = e4m3x8_to_bf16x8_scaled(c[0], c[1], e), hi = e4m3x8_to_bf16x8_scaled(c[2], c[3], e);
#pragma unroll
            for (int f = 0; f < 2; ++f)
              part[f][lo_at] = mfma_bf16(lo, __builtin_bit_cast(bf16x8, qf[f][2 * j]), part[f][lo_at]);
#pragma unroll
            for (int f = 0; f < 2; ++f)
              part[f][hi_at] = mfma_bf16(hi, __builtin_bit_cast(bf16x8, qf[f][2 * j + 1]), part[f][hi_at]);
          } else {
            constexpr int to = KT == 2 ? k : j & 1;
#pragma unroll
            for (int f = 0; f < 2; ++f) part[f][to] = mfma_bf16_16x16x32(c, qf[f][F8 ? j + 8 : j], part[f][to]);
          }
          if constexpr (i % kFence == kFence - 1) __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          if constexpr (KT == 2) {
            sc[0][f] = part[f][0];
            sc[KT - 1][f] = part[f][1];
          } else {
            sc[0][f] = part[f][0] + part[f][1];
          }
        }
        __builtin_amdgcn_sched_barrier(0);

        // ---- masks: only where the step passes what some row sees, or misses a page
        const uint32_t have = (uint32_t)uniform(valid) >> (8 * wk * KT);
        if ((u + 1) * M::kStep > pc.see_all || (have & (KT == 2 ? 0x0101u : 1u)) != (KT == 2 ? 0x0101u : 1u)) {
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int k = 0; k < KT; ++k) {
              const int upto = (have >> (8 * k)) & 1 ? sees[f] - (u * M::kStep + (wk * KT + k) * 16 + 4 * g) : 0;
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[k][f][i] = i < upto ? sc[k][f][i] : -INFINITY;
            }
        }
        bool move = false;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          float top = sc[0][f][0];
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[k][f][i]);
          top = rows_max(top) * scale_log2;
          move = move || top > m[f] + kLazy;  // from -inf: any finite score
          if (g == 0) tops[wk * MR + (wq * 2 + f) * 16 + r16] = top;
        }
        const bool any = __any(move);
        if (lane == 0) lds[M::kFlags + (u & 1) * 4 + wave] = any ? 1 : 0;
        put_p(u);
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        float sum = l[f];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int q = (wq * 2 + f) * 16 + r16;
        if (g == 0) fin[wk * MR + q] = sum;
        if (wk == 0 && g == 0) fin[2 * MR + q] = m[f];
      }
      lds_barrier();
    }
  } else {
    // ================ output, and the loads
    const int w = wave - 4;
    constexpr int CT = 8, RG = M::kGroups;
    int load_off[L::kLoads];  // source bytes within a group of 8 rows; the swizzle differs in odd groups
#pragma unroll
    for (int j = 0; j < L::kLoads; ++j) {
      const int slot = j * 64 + lane, row = slot / L::kChunks, pos = slot % L::kChunks;
      load_off[j] = row * L::kRowB + ((pos ^ swz(RG == 1 ? (w & 1) * 8 + row : row)) << 4);
    }
    while (cur < uniform(side->end)) {
      Piece pc;
      const bool there = next_piece<MR>(place, side, cur, &pc);
      cur += pc.s1 - pc.s0;
      if (!there) continue;
      const int u0 = pc.s0 * (64 / M::kStep);
      const int end = min(pc.s1 * (64 / M::kStep), (pc.see_any + M::kStep - 1) / M::kStep);

      // Where the wave's 16-row block stands in steps held .. held + 63, a lane each.
      const int32_t* table = in.pages.table + (long long)pc.b * in.pages.max_pages;
      int held = u0, where;
      const auto look_up = [&]() __attribute__((always_inline)) {
        where = find_block(in.pages, table, min(held + lane, end - 1) * (M::kStep / 16) + w * RG / 2);
      };
      look_up();
      const uint8_t* src;
      const uint32_t* src_scales;
      uint32_t dst, dst_scales;
      const auto aim = [&](int u) __attribute__((always_inline)) {
        if (u == held + 64) {
          held = u;
          look_up();
        }
        const int at = __builtin_amdgcn_readlane(where, u - held), buffer = u % M::kBufs;
        const long long row = (at >= 0 ? (long long)at << 4 : 0) + (RG == 1 ? (w & 1) * 8 : 0);  // no page: some row, masked
        if (lane == 0) lds[M::kValid + buffer * 4 + w * RG / 2] = at >= 0 ? 1 : 0;
        src = a.data + row * L::kRowB;
        dst = uniform(lds_address(lds) + buffer * M::kBytes + w * RG * 8 * L::kRowB);
        if constexpr (F8) {
          src_scales = a.scales + row;
          dst_scales = uniform(lds_address(lds) + buffer * M::kBytes + M::kData + w * RG * 32);
        }
      };
      const auto load = [&](int i) __attribute__((always_inline)) {
        if (F8 && i == M::kLoad - 1) {
          if (lane < RG * 8) dma_4(src_scales, lane * 4, dst_scales);
        } else if (i < L::kLoads) {
          dma_16(src, load_off[i], dst + i * 1024);
        } else {
          dma_16(src + 8 * L::kRowB, load_off[i - L::kLoads] ^ 64, dst + 8 * L::kRowB + (i - L::kLoads) * 1024);
        }
      };
      const auto load_all = [&](int u) __attribute__((always_inline)) {
        if (u < end) {
          aim(u);
#pragma unroll
          for (int j = 0; j < M::kLoad; ++j) load(j);
        }
      };
      // Step u has landed; the steps after it may be on their way.
      const auto landed = [&](int u) __attribute__((always_inline)) {
        if (M::kAway == 2 && u + 1 < end) wait_vmcnt<M::kLoad>();
        else wait_vmcnt<0>();
      };
      f32x4 o[CT][4];
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][f] = f32x4{0.f, 0.f, 0.f, 0.f};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < M::kAway; ++i) load_all(u0 + i);
      __builtin_amdgcn_sched_barrier(0);

      if (end > u0) {  // the first step has its scores taken
        landed(u0);
        lds_barrier();
        load_all(u0 + M::kAway);
      }
      for (int u = u0 + 1; u <= end; ++u) {
        landed(u);
        lds_barrier();  // step u has landed, P of step v is there, and the step before that is done with
        const int v = u - 1, buffer = v % M::kBufs;  // the step that is added
        // ---- O^T += V^T P^T: lane (column r16, key octet g).  What is read first goes
        // out before anything is waited for.
        const int flags = *reinterpret_cast<const int*>(lds + M::kFlags + (v & 1) * 4);
        const uint32_t valid = *reinterpret_cast<const uint32_t*>(lds + M::kValid + buffer * 4);
        const uint8_t* pbuf = lds + M::kP + (v & 1) * M::kPBytes + r16 * M::kPRow;
        u32x4 p[4];
        u32x4 words[2];
        const auto get_p = [&](int h) __attribute__((always_inline)) {
          if constexpr (F8) {
            const uint8_t* from = lds + buffer * M::kBytes + M::kData + (h * 32 + 8 * g) * 4;
            words[0] = ld_u32x4(from);
            words[1] = ld_u32x4(from + 16);
          }
#pragma unroll
          for (int f = 0; f < 4; ++f) p[f] = ld_u32x4(pbuf + f * 16 * M::kPRow + (((4 * h + g) ^ zp) << 4));
        };
        get_p(0);
        load_all(u + M::kAway);  // at once: between the products they held the wave up for longer
        if (uniform(flags) != 0) {
          lds_barrier();
          get_p(0);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float by = tops[2 * MR + f * 16 + r16];
#pragma unroll
            for (int c = 0; c < CT; ++c) o[c][f] *= by;
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        uint8_t* buf = lds + buffer * M::kBytes;
        constexpr uint32_t kAll = M::kStep == 64 ? 0x01010101u : 0x0101u;
        const uint32_t ok = (uint32_t)uniform(valid) & kAll;
        const bool edge = (v + 1) * M::kStep > pc.see_all || ok != kAll;
        if (edge) {
          clear_unseen<F8, M::kStep>(in, pc, buf, v * M::kStep, ok, w * (F8 ? 8 : 16), o);
          asm volatile("" ::: "memory");
        }
        __builtin_amdgcn_sched_barrier(0);

        // An exclusive-or of the block into the address is the swizzle.
        const int row = 8 * g + (F8 ? r16 >> 1 : r16 >> 2);
        const uint32_t at = (uint32_t)buffer * M::kBytes + row * L::kRowB + w * (F8 ? 128 : 256) +
                            ((swz(row) ^ (F8 ? 0 : (lane >> 1) & 1)) << 4) + 8 * (lane & 1);
        constexpr int NF = M::kStep / 32 * CT;
        const auto frag = [&](int i) {  // i = (half, block)
          const int h = i / CT, c = i % CT;
          if constexpr (F8) {
            const u32x2 x = lds_tr8(lds + (at ^ (c << 4)) + h * 32 * L::kRowB);
            return u32x4{x[0], x[1], 0u, 0u};
          } else {  // rows 4 further: bits 0 and 2 of the swizzle flip
            const u32x2 x0 = lds_tr16(lds + (at ^ ((c & 3) << 5)) + (c >> 2) * 128);
            const u32x2 x1 = lds_tr16(lds + (at ^ ((c & 3) << 5) ^ 80) + (c >> 2) * 128 + 4 * L::kRowB);
            return u32x4{x0[0], x0[1], x1[0], x1[1]};
          }
        };
        u32x4 ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = frag(i);
        // e4m3: a probability takes its key's power of two for the wave's columns, by adding
        // to the exponents of two at a time: 121.5 us for chunks of 200 and 500 tokens on 3500
        // and 5000 keys, 125.7 by widening, two products and rounding.  Exact for normal numbers; a
        // product below 2^-126 becomes some number below 2^-126.  Zeros stay zeros (P is zero
        // or normal): a key that a query does not see, or whose term vanished, may have any scale.
        // The pair of ones is kept from the compiler, which would make compares and selects of
        // the minimum's product (8% more time).
        uint32_t ones = 0x00010001u;
        if constexpr (F8) asm("" : "+s"(ones));
        const auto scale_p = [&](int h) __attribute__((always_inline)) {
          if constexpr (F8) {
            u16x2 add[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t w0 = words[i >> 1][2 * (i & 1)] >> (8 * w), w1 = words[i >> 1][2 * (i & 1) + 1] >> (8 * w);
              add[i] = __builtin_bit_cast(u16x2, (w0 & 255u) | (w1 & 255u) << 16) * (uint16_t)128 - (uint16_t)(127 * 128);
            }
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t pair = p[f][i];
                const u16x2 from = __builtin_bit_cast(u16x2, pair);
                const u16x2 sum = add[i] * __builtin_elementwise_min(from, __builtin_bit_cast(u16x2, ones)) + from;
                p[f][i] = __builtin_bit_cast(uint32_t,
                                             __builtin_elementwise_max(__builtin_bit_cast(s16x2, sum), s16x2{0, 0}));
              }
          }
        };
        scale_p(0);
        static_for<0, NF>([&](auto ic) {
          constexpr int i = decltype(ic)::value, c = i % CT, h = i / CT;
          const u32x4 x = ring[i % kAhead];
          if constexpr (i + kAhead < NF) ring[i % kAhead] = frag(i + kAhead);
          const bf16x8 xb = F8 ? e4m3x8_to_bf16x8(x[0], x[1]) : __builtin_bit_cast(bf16x8, x);
#pragma unroll
          for (int f = 0; f < 4; ++f) o[c][f] = mfma_bf16(xb, __builtin_bit_cast(bf16x8, p[f]), o[c][f]);
          if constexpr (i % 2 == 1) {
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (c == CT - 1 && h + 1 < M::kStep / 32) {
            get_p(h + 1);
            scale_p(h + 1);
            __builtin_amdgcn_sched_barrier(0);
          }
        });
      }
      lds_barrier();  // sums and maxima
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int q = f * 16 + r16;
        put_rows<MR>(side, pc, f, r16, w * 128 + 4 * g, w == 0 && g == 0, fin[2 * MR + q], fin[q] + fin[MR + q], o);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// Joins the pieces of the query rows that were cut, in the order of the keys.

// The record of a row; false where nothing is to be joined.
__device__ __forceinline__ bool to_join(const Args& a, int mr, long long row, LatentRecord* where, int* r) {
  const int4 rec = a.rows()[row];  // rows behind the last sequence have none: whatever stands there
  *where = LatentRecord{rec.x, rec.y};
  *r = rec.z;
  return row >= (long long)max(a.cu_q[0], 0) * a.H && row < (long long)min(a.cu_q[a.B], a.T) * a.H &&
         latent_record_joins(*where, a.side_by_side) && (unsigned)rec.z < (unsigned)mr;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// A piece's weight and part of the sum.  l may be NaN where the maximum is -inf (a NaN
// that is a piece's only key), and the row is NaN then.
__device__ __forceinline__ float piece_weight(float2 v, float base) { return __builtin_amdgcn_exp2f(v.x - base); }
__device__ __forceinline__ float piece_sum(float2 v, float base) {
  return v.y != 0.f ? v.y * piece_weight(v, base) : 0.f;
}

// Many rows, few pieces each: a wave per row, 8 columns per lane, the pieces' weights
// 64 at a time in the lanes, four pieces' loads under way together.
__global__ __launch_bounds__(256) void latent_join_kernel(Args a, int mr, int rows) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  LatentRecord where;
  int r;
  if (!to_join(a, mr, row, &where, &r)) return;
  const float2* ml = a.ml();
  const float* part = a.part(mr) + lane * 4;
  const auto at = [&](int j) { return (long long)latent_record_slot(where, a.side_by_side, j) * mr + r; };
  // The first pieces' outputs come under their maxima, four pieces at a time: 71 registers
  // leave room for seven waves per SIMD (chunks of 200 to 500 tokens: 2% less time for the
  // whole call than with eight at a time, after the maxima).
  f32x4 x[4][2];
  const auto load = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* from = part + at(min(j + i, where.pieces - 1)) * kLatent;  // past the last: again, unused
      x[i][0] = *reinterpret_cast<const f32x4*>(from);
      x[i][1] = *reinterpret_cast<const f32x4*>(from + 256);
    }
  };
  load(0);
  float top = -INFINITY;
  float2 v = lane < where.pieces ? ml[at(lane)] : make_float2(-INFINITY, 0.f);
  top = v.x;
  for (int j = lane + 64; j < where.pieces; j += 64) top = fmaxf(top, ml[at(j)].x);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  float sum = 0.f, w = 0.f;
  for (int j = 0; j < where.pieces; j += 4) {
    if (j % 64 == 0) {
      if (j > 0) v = j + lane < where.pieces ? ml[at(j + lane)] : make_float2(-INFINITY, 0.f);
      sum += piece_sum(v, base);
      w = piece_weight(v, base);
    }
    if (j > 0) load(j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float wi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j % 64 + i));
      if (j + i < where.pieces) {
        acc[0] += x[i][0] * wi;
        acc[1] += x[i][1] * wi;
      }
    }
  }
  sum = wave_add(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *reinterpret_cast<u32x2*>(a.out + (long long)row * kLatent + h * 256 + lane * 4) =
        u32x2{pack_bf16x2(acc[h][0] * inv, acc[h][1] * inv), pack_bf16x2(acc[h][2] * inv, acc[h][3] * inv)};
  if (a.lse != nullptr && lane == 0)
    a.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Few rows, up to kUnits pieces each: a work-group per row and 128 columns, 32 lanes
// across and the pieces dealt to 8 groups of lanes, 8 in flight each.  A wave per row /
// this, whole call, us: 16 heads, e4m3, one sequence of 100001 69.4 / 28.2, 16 of 6000 28.7 /
// 27.6, 32 of 6000 (512 rows) 40.1 / 40.3, 64 of 600 to 8000 (1024 rows) 50.4 / 53.1.
__global__ __launch_bounds__(256) void latent_join_long_kernel(Args a, int mr) {
  constexpr int ACROSS = 32, GROUPS = 256 / ACROSS;
  __shared__ f32x4 red[256];
  __shared__ float weight[kUnits], stat[8];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  LatentRecord where;
  int r;
  if (!to_join(a, mr, row, &where, &r)) return;
  const int across = threadIdx.x % ACROSS, group = threadIdx.x / ACROSS, col = (blockIdx.y * ACROSS + across) * 4;
  const auto at = [&](int j) { return (long long)latent_record_slot(where, a.side_by_side, j) * mr + r; };
  const float2 v = (int)threadIdx.x < where.pieces ? a.ml()[at(threadIdx.x)] : make_float2(-INFINITY, 0.f);
  const float* part = a.part(mr) + col;
  f32x4 x[8];
  const auto load = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = j0 + group + GROUPS * i;
      x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (j < where.pieces) x[i] = *reinterpret_cast<const f32x4*>(part + at(j) * kLatent);
    }
  };
  load(0);  // under the weights
  float top = wave_max(v.x);
  if (lane == 0) stat[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = wave_add(piece_sum(v, base));
  weight[threadIdx.x] = piece_weight(v, base);
  if (lane == 0) stat[4 + wave] = sum;
  __syncthreads();
  sum = (stat[4] + stat[5]) + (stat[6] + stat[7]);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0;;) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc += x[i] * weight[j0 + group + GROUPS * i];
    j0 += 8 * GROUPS;
    if (j0 >= where.pieces) break;
    load(j0);
  }
  red[threadIdx.x] = acc;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) acc += red[i * ACROSS + across];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<u32x2*>(a.out + (long long)row * kLatent + col) =
      u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  if (a.lse != nullptr && col == 0)
    a.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

int launch_join(const Args& a, int mr, hipStream_t st) {
  const unsigned rows = (unsigned)((long long)a.T * a.H);
  if (rows <= kJoinRows)
    hipLaunchKernelGGL(latent_join_long_kernel, dim3(rows, kLatent / 128), dim3(256), 0, st, a, mr);
  else
    hipLaunchKernelGGL(latent_join_kernel, dim3((rows + 3) / 4), dim3(256), 0, st, a, mr, (int)rows);
  return (int)hipGetLastError();
}

template <int WQ, int WK, bool F8>
int launch(const Args& a, hipStream_t st) {
  constexpr int mr = 16 * WQ, lds = Lds<mr, WK, F8>::kBytes;
  FERRET_HIP_CHECK((set_lds_limit_once<latent_attention_kernel<WQ, WK, F8>>(lds)));
  hipLaunchKernelGGL((latent_attention_kernel<WQ, WK, F8>), dim3(kUnits), dim3(64 * WQ * WK), lds, st, a);
  FERRET_HIP_CHECK(hipGetLastError());
  return launch_join(a, mr, st);
}

template <bool F8>
int launch_wide(const Args& a, hipStream_t st) {
  constexpr int lds = Wide<F8>::kLds;
  FERRET_HIP_CHECK((set_lds_limit_once<latent_attention_wide_kernel<F8>>(lds)));
  hipLaunchKernelGGL((latent_attention_wide_kernel<F8>), dim3(kUnits), dim3(512), lds, st, a);
  FERRET_HIP_CHECK(hipGetLastError());
  return launch_join(a, Wide<F8>::kRows, st);
}

template <bool F8>
int launch_rows(int mr, const Args& a, hipStream_t st) {
  switch (mr) {
    case 16: return launch<1, 4, F8>(a, st);
    case 32: return launch<2, 4, F8>(a, st);
    default: return launch_wide<F8>(a, st);
  }
}

// Query rows per tile by the rows that a sequence has on average.  Us, e4m3, 64 sequences
// of 3000: 32 heads 46.9 in tiles of 32, 56.7 of 16, 48.7 of 64; 16 heads of 600 to 8000
// 50.4 of 16, 54.6 of 32; 32 of 3000, 64 heads 39.8 of 64, 45.3 of 32; 128 heads, bf16,
// 32 of 900 to 6000 58.8 of 64 against 80.6 of 32.
int tile_rows(int T, int B, int H) {
  const long long rows = (long long)T * H / B;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

// Row tiles side by side by the tiles that a sequence has on average: work-groups of one
// XCD that walk the same keys at the same time.  128 heads (two tiles), bf16, 32 sequences of
// 900 to 6000: 58.8 us two at a time, 66.0 one after another, 79.9 four; 500 new tokens of
// two sequences of 4000, 16 heads, e4m3: 138 us eight at a time, 139 two, 158 one.
int side_by_side(int T, int B, int H) {
  const long long tiles = (long long)T * H / B / 64;
  return tiles < 2 ? 1 : tiles < 4 ? 2 : tiles < 8 ? 4 : 8;
}

}  // namespace
}  // namespace ferret

using namespace ferret;

int ferret_check_pages(const int32_t* page_table, int B, int max_pages, int pages, int page_size);

extern "C" size_t ferret_latent_attention_workspace(int B, int T, int H) {
  if (B < 1 || T < 1 || H < 1 || (long long)T * H >= (1LL << 31)) return 0;
  const size_t mr = tile_rows(T, B, H), rows = ((size_t)T * H * sizeof(int4) + 255) & ~(size_t)255;
  return rows + 2 * kUnits * mr * (sizeof(float2) + kLatent * sizeof(float));
}

extern "C" int ferret_latent_attention(const void* q_latent, long long ql_token, long long ql_head,
                                       const void* q_rotary, long long qr_token, long long qr_head, const void* data,
                                       const void* scales, int pages, int page_size, const int32_t* page_table,
                                       const int32_t* lens, const int32_t* cu_q, int B, int max_pages, int T, int H,
                                       float scale, int causal, void* out, float* lse, void* ws, size_t ws_bytes,
                                       void* stream) {
  FERRET_REQUIRE(q_latent && q_rotary && data && lens && cu_q && out, FERRET_ERR_NULL);
  const int rc = ferret_check_pages(page_table, B, max_pages, pages, page_size);
  if (rc != FERRET_OK) return rc;
  FERRET_REQUIRE(T >= 1 && H >= 1 && H <= 1024 && (long long)T * H < (1LL << 31), FERRET_ERR_SHAPE);
  FERRET_REQUIRE(scale > 0.f && scale < 1e30f, FERRET_ERR_SHAPE);
  for (const long long stride : {ql_token, ql_head, qr_token, qr_head})
    FERRET_REQUIRE(stride >= 0 && stride < (1LL << 31), FERRET_ERR_SHAPE);
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE(((bits(q_latent) | bits(q_rotary) | bits(data) | bits(out)) & 15) == 0 &&
                     ((bits(scales) | bits(lse)) & 3) == 0 && ((ql_token | ql_head | qr_token | qr_head) & 7) == 0,
                 FERRET_ERR_ALIGN);
  const int mr = tile_rows(T, B, H);
  FERRET_REQUIRE((long long)max_pages * page_size <= (1LL << 31) - 2 * kKeys, FERRET_ERR_SHAPE);  // a step's end stays below 2^31
  // steps of the whole batch are counted in 32 bits, rounded up to whole shares
  FERRET_REQUIRE((long long)pages * page_size < (1LL << 35), FERRET_ERR_SHAPE);
  const long long tiles = (long long)T * H / mr + B, most = ((long long)max_pages * page_size + kKeys - 1) / kKeys + kLatentExtra;
  FERRET_REQUIRE(tiles * most < (1LL << 31) - kUnits, FERRET_ERR_SHAPE);
  const size_t need = ferret_latent_attention_workspace(B, T, H);
  FERRET_REQUIRE(ws != nullptr && ws_bytes >= need && (bits(ws) & 15) == 0, FERRET_ERR_WORKSPACE);
  // In place is sound: the work-group that has read a whole tile writes it, the join those
  // that were cut.
  const bool over = in_place(out, q_latent, T, ql_token, H, ql_head, kLatent);
  FERRET_REQUIRE(!clash({Range{out, (uint64_t)T * H * kLatent * 2}, Range{lse, (uint64_t)T * H * 4}, Range{ws, need}},
                        {bf16_range(over ? nullptr : q_latent, T, ql_token, H, ql_head, kLatent),
                         bf16_range(q_rotary, T, qr_token, H, qr_head, kRotary),
                         data_range(data, scales, pages, page_size), scale_range(scales, pages, page_size),
                         ints_range(page_table, (uint64_t)B * max_pages), ints_range(lens, B),
                         ints_range(cu_q, B + 1LL)}),
                 FERRET_ERR_SHAPE);
  Args a;
  a.ql = static_cast<const uint16_t*>(q_latent);
  a.qr = static_cast<const uint16_t*>(q_rotary);
  a.ql_t = (int)ql_token;
  a.ql_h = (int)ql_head;
  a.qr_t = (int)qr_token;
  a.qr_h = (int)qr_head;
  a.data = static_cast<const uint8_t*>(data);
  a.scales = static_cast<const uint32_t*>(scales);
  a.pages = Pages{page_table, max_pages, pages, page_size};
  a.lens = lens;
  a.cu_q = cu_q;
  a.B = B;
  a.T = T;
  a.H = H;
  a.scale_log2 = scale * kLog2e;
  a.causal = causal != 0;
  // Shares of one step where a step is short: 16 heads, 256 keys 13.2 us against 14.8 in
  // shares of two; 128 heads, e4m3, 8 sequences of 100 keys 20.4 in shares of two, 21.0 of one.
  a.min_steps = mr == 64 ? 2 : 1;
  a.side_by_side = side_by_side(T, B, H);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.ws = static_cast<uint8_t*>(ws);
  return scales != nullptr ? launch_rows<true>(mr, a, (hipStream_t)stream)
                           : launch_rows<false>(mr, a, (hipStream_t)stream);
}
