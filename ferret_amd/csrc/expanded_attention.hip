// Latent attention in its expanded form: ragged prompts over per-head keys and values
// (128 + 64 and 128 wide), the 64 rotary key values shared by all heads:
//   s_ij = scale * (qn_i . kn_j + qr_i . kr_j),   o_i = sum_j softmax_j(s_ij) v_j
// for one head; token i of n new ones sees the keys j <= len - n + i of its sequence
// (causal) or all len.  A token that sees none gives zeros and lse -inf.
//
// A work-group takes 128 tokens of one head, 32 per wave, and walks the keys in steps of
// 64.  Either one team of four waves walks them all and two work-groups share a CU, or
// two teams take steps in turn and join their outputs at the end.  Both put two waves on
// each SIMD, so that one's softmax runs under the other's products, and both fill the
// 160 KB of a CU; two teams halve the time of a long tile, one needs no join.  Where
// there are fewer tiles than CUs, parts of a tile's keys go to work-groups of their own
// (two teams each), whose fp32 partials a second kernel joins in order.  Keys and
// values come into LDS by asynchronous loads, one step ahead.  S^T = K Q^T has the keys
// as MFMA rows: a lane holds the scores of one query and, per block, four consecutive
// keys, which is the operand that O^T = V^T P^T needs (the order of the keys within the
// contraction is free as long as V^T follows it), so P never leaves its registers.  V^T
// comes from row-major V by transposing LDS reads.  Tiles go longest first
// (expanded_plan.hpp), and a head's tiles to one XCD where the number of heads is a
// multiple of 8 (keys from its L2).
//
// Bound by the matrix and vector pipes together: 2 * (192 + 128) operations per query,
// visible key and head keep the first busy for 52% of a long prompt's cycles,
// exponentials, packing and masks the second for 36% or more, at a clock that falls
// below 2 GHz; no LDS bank conflicts.
// 16 heads, 4096 new tokens after 4096 others: 240 us, 1070 TFLOP/s (counting visible
// pairs), where a large product of the library reaches 1206.  S, m, l and O are fp32; P is
// rounded to bf16 (half a step, 2^-8 relative), l sums the unrounded terms.
#include "attention.hpp"
#include "expanded_plan.hpp"
#include "ranges.hpp"

#include <algorithm>
#include <initializer_list>

namespace ferret {
namespace {

constexpr int kNope = 128, kRope = 64, kValue = 128;
constexpr int kStep = kTileKeys, kTokens = kTileTokens;
constexpr int kKn = 0, kKr = kStep * kNope * 2;        // a buffer: keys, rotary keys, values
constexpr int kV = kKr + kStep * kRope * 2, kBuf = kV + kStep * kValue * 2;
static_assert(4 * kBuf <= 160 * 1024, "LDS of a CU: two work-groups, or one of two teams");

// Key and value fragments are read ahead of their products in rings that scheduling
// fences keep: 4096 after 4096 others, in one team: 240.2 us, 3% less than where the
// compiler places the reads, two at a time; 4 and 4, or 8 and 4, with a fence per 4
// products: 240.6 and 240.0.
constexpr int kAheadK = 6, kAheadV = 4, kFence = 2;
constexpr int kCus = 256;
constexpr int kMaxParts = 16, kPartSteps = 6;

// Bytes of the maxima and sums of so many rows: the outputs behind them are read 16 bytes at a time.
__host__ __device__ constexpr size_t stat_bytes(size_t rows) { return (rows * sizeof(float2) + 15) & ~(size_t)15; }

struct Args {
  const uint16_t *qn, *qr, *kn, *kr, *v;
  int qn_t, qn_h, qr_t, qr_h, kn_s, kn_h, kr_s, v_s, v_h;  // strides in elements
  const int32_t *cu_q, *cu_k;
  int B, T, S, H;
  float scale_log2;
  int causal;
  uint16_t* out;  // [T, H, 128]
  float* lse;     // [T, H] or null
  int parts;      // of a tile's keys
  float2* ml;     // [parts][T * H]: maxima and sums, then on a 16-byte bound the outputs [parts][T * H][128]
  __host__ __device__ float* part() const {
    return reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ml) + stat_bytes((size_t)parts * T * H));
  }
};

// The swizzles: 16-byte chunk c of row r stands at c ^ swizzle(r).  Rows of 256
// bytes (a whole turn of the banks) and of 128.
__device__ __forceinline__ int swz_kn(int r) { return r & 15; }
__device__ __forceinline__ int swz_kr(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz_v(int r) { return 2 * (r & 7); }

// Index values outside the tensors are cut to them.
__device__ __forceinline__ TileSeq tiles_of(const Args& a, int b) {
  const int q0 = min(max(a.cu_q[b], 0), a.T), k0 = min(max(a.cu_k[b], 0), a.S);
  return TileSeq{min(max(a.cu_q[b + 1], q0), a.T) - q0, min(max(a.cu_k[b + 1], k0), a.S) - k0, a.causal};
}

template <int TEAMS, bool SPLIT>
__global__ __launch_bounds__(256 * TEAMS, 2) void expanded_attention_kernel(Args a) {
  constexpr int QF = 2, KT = kStep / 16, CT = kValue / 16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6) & 3, team = TEAMS == 2 ? uniform(threadIdx.x >> 8) : 0;
  const int r16 = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.H;

  // ---- the tile: every wave finds it by itself
  int b = -1, tile = 0;
  const int in_line = blockIdx.x / a.H, slot = SPLIT ? in_line / a.parts : in_line;
  if (a.B <= kOrderedBatch) {
    // The longest tiles of the batch first: the length of the rank-th, 64 lengths at a
    // time, a lane each; then the tile among those of that length.
    const TileSeq mine = lane < a.B ? tiles_of(a, lane) : TileSeq{0, 0, 0};  // one load deep
    const auto seq = [&](int i) __attribute__((always_inline)) {
      return TileSeq{__builtin_amdgcn_readlane(mine.n, i), __builtin_amdgcn_readlane(mine.len, i), a.causal};
    };
    int all = 0;
    for (int i = 0; i < a.B; ++i) all += seq(i).tiles();
    if (slot >= all) return;
    const int rank = TEAMS == 2 ? slot : paired_rank(slot, all, kCus / a.H);
    int base = 0, stride = (a.S + kStep - 1) / kStep / 64 + 1;
    for (;;) {
      int count = 0;
      for (int i = 0; i < a.B; ++i) count += seq(i).at_least(base + lane * stride);
      const unsigned long long enough = __ballot(count > rank);
      base += (63 - __clzll((long long)enough)) * stride;  // lane 0's are enough
      if (stride == 1) break;
      stride = (stride + 63) / 64;
    }
    int before = 0;
    for (int i = 0; i < a.B; ++i) before += seq(i).at_least(base + 1);
    int among = rank - before;
    for (int i = 0; i < a.B && b < 0; ++i) {
      const TileSeq s = seq(i);
      const int from = s.first_of(base), count = s.first_of(base + 1) - from;
      if (among < count) {
        b = i;
        tile = from + among;
      }
      among -= count;
    }
  } else {
    // Sequence by sequence, each from its longest tile on.
    int left = slot;
    for (int base = 0; base < a.B; base += 64) {
      const int tiles = base + lane < a.B ? tiles_of(a, base + lane).tiles() : 0;
      int incl = tiles;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
      }
      const unsigned long long past = __ballot(left < incl);
      if (past != 0) {
        const int at = __ffsll((long long)past) - 1;
        b = base + at;
        const int count = __shfl(tiles, at, 64), before = __shfl(incl, at, 64) - count;
        tile = count - 1 - (left - before);
        break;
      }
      left -= __shfl(incl, 63, 64);
    }
  }
  b = uniform(b);
  if (b < 0) return;
  const int q0 = uniform(min(max(a.cu_q[b], 0), a.T));
  const int n = uniform(min(max(a.cu_q[b + 1], q0), a.T)) - q0;
  const int k0 = uniform(min(max(a.cu_k[b], 0), a.S));
  const int len = uniform(min(max(a.cu_k[b + 1], k0), a.S)) - k0;
  const int row0 = uniform(tile) * kTokens, row_last = min(row0 + kTokens, n) - 1;
  const int past = len - n + 1;
  const int see_all = a.causal ? max(past + row0, 0) : len;        // keys of the first token
  const int see_any = a.causal ? max(past + row_last, 0) : len;    // and of the last
  const int steps = (min(see_any, len) + kStep - 1) / kStep;
  const int part = SPLIT ? uniform(in_line - slot * a.parts) : 0;
  const int share = SPLIT ? (steps + 2 * a.parts - 1) / (2 * a.parts) * 2 : steps;  // whole turns of both teams
  const int first = part * share, last = min(first + share, steps);

  // ---- steps into LDS: this wave's 16 rows of each array (4, 8 and 4 rows per load).
  // The team takes steps team, team + TEAMS, ...
  uint8_t* const own = lds + team * 2 * kBuf;
  const uint8_t* kn = reinterpret_cast<const uint8_t*>(a.kn + (long long)k0 * a.kn_s + (long long)head * a.kn_h);
  const uint8_t* kr = reinterpret_cast<const uint8_t*>(a.kr + (long long)k0 * a.kr_s);
  const uint8_t* vv = reinterpret_cast<const uint8_t*>(a.v + (long long)k0 * a.v_s + (long long)head * a.v_h);
  const auto issue = [&](int t) {
    const uint32_t buf = uniform(lds_address(own) + (t / TEAMS & 1) * kBuf);
    const int most = len - 1 - t * kStep;  // rows past the sequence repeat its last one
    const uint8_t* kn_t = kn + (long long)t * kStep * a.kn_s * 2;
    const uint8_t* kr_t = kr + (long long)t * kStep * a.kr_s * 2;
    const uint8_t* v_t = vv + (long long)t * kStep * a.v_s * 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = wave * 16 + j * 4 + g;
      dma_16(kn_t, min(r, most) * a.kn_s * 2 + ((r16 ^ swz_kn(r)) << 4), buf + kKn + (wave * 16 + j * 4) * 256);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = wave * 16 + j * 8 + (lane >> 3);
      dma_16(kr_t, min(r, most) * a.kr_s * 2 + (((lane & 7) ^ swz_kr(r)) << 4), buf + kKr + (wave * 16 + j * 8) * 128);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = wave * 16 + j * 4 + g;
      dma_16(v_t, min(r, most) * a.v_s * 2 + ((r16 ^ swz_v(r)) << 4), buf + kV + (wave * 16 + j * 4) * 256);
    }
  };
  if (first + team < last) issue(first + team);

  // ---- queries (rows past the tile's repeat its last one)
  u32x4 qf[QF][6];
  int sees[QF];
#pragma unroll
  for (int f = 0; f < QF; ++f) {
    const int r = row0 + (wave * QF + f) * 16 + r16, rc = min(r, row_last);
    sees[f] = r <= row_last ? min(max(a.causal ? past + r : len, 0), len) : 0;
    const uint16_t* qn = a.qn + (long long)(q0 + rc) * a.qn_t + (long long)head * a.qn_h;
    const uint16_t* qr = a.qr + (long long)(q0 + rc) * a.qr_t + (long long)head * a.qr_h;
#pragma unroll
    for (int k = 0; k < 4; ++k) qf[f][k] = ld_u32x4(qn + 32 * k + 8 * g);
#pragma unroll
    for (int k = 0; k < 2; ++k) qf[f][4 + k] = ld_u32x4(qr + 32 * k + 8 * g);
  }
  wait_vmcnt<0>();
  __builtin_amdgcn_sched_barrier(0);

  f32x4 o[CT][QF];
  float m[QF], l[QF];
#pragma unroll
  for (int f = 0; f < QF; ++f) {
    m[f] = -INFINITY;
    l[f] = 0.f;
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (int turn = first; turn < last; turn += TEAMS) {
    const int t = turn + team;
    const bool live = TEAMS == 1 || t < last;
    wait_vmcnt<0>();
    lds_barrier();  // the steps have landed for every wave, and the other buffers have been read
    if (t + TEAMS < last) issue(t + TEAMS);
    __builtin_amdgcn_sched_barrier(0);
    const int buffer = (team * 2 + (t / TEAMS & 1)) * kBuf;
    uint8_t* buf = lds + buffer;

    // ---- S^T: 16 keys x 16 queries per block
    f32x4 sc[KT][QF];
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int f = 0; f < QF; ++f) sc[k][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (live) {
      const uint8_t* nope = buf + kKn + r16 * 256;
      const uint8_t* rope = buf + kKr + r16 * 128;
      const int zn = (g ^ (r16 & 3)) << 4, zr = (g ^ (swz_kr(r16) & 3)) << 4;
      const auto frag = [&](int i) __attribute__((always_inline)) {  // i = (block, chunk)
        const int k = i / 6, j = i % 6;
        return j < 4 ? ld_u32x4(nope + k * 16 * 256 + (zn | ((j ^ (r16 >> 2)) << 6)))
                     : ld_u32x4(rope + k * 16 * 128 + (zr | (((j - 4) ^ (swz_kr(r16) >> 2)) << 6)));
      };
      u32x4 ring[kAheadK];
#pragma unroll
      for (int i = 0; i < kAheadK; ++i) ring[i] = frag(i);
      static_for<0, KT * 6>([&](auto ic) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value, k = i / 6, j = i % 6;
        const u32x4 c = ring[i % kAheadK];
        if constexpr (i + kAheadK < KT * 6) ring[i % kAheadK] = frag(i + kAheadK);
#pragma unroll
        for (int f = 0; f < QF; ++f) sc[k][f] = mfma_bf16_16x16x32(c, qf[f][j], sc[k][f]);
        if constexpr (i % kFence == kFence - 1) __builtin_amdgcn_sched_barrier(0);
      });
    }

    // ---- masks: only where the step passes what some token of the tile sees
    unsigned long long odd = 0;  // rows with Inf or NaN among the values that not all tokens see
    if ((turn + TEAMS) * kStep > see_all) {  // of either team: the barriers are for both
#pragma unroll
      for (int f = 0; f < QF; ++f) {
        const int upto = sees[f] - t * kStep - 4 * g;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[k][f][i] = k * 16 + i < upto ? sc[k][f][i] : -INFINITY;
      }
      // Values that a token does not see must not reach it as 0 * NaN: rows that no
      // token sees become zeros; Inf and NaN of rows that some see are cleared and
      // added below to those that do.  The record of such rows takes the keys' place.
      lds_barrier();  // the keys have been read
      unsigned* found = reinterpret_cast<unsigned*>(buf + kKn);
      if ((threadIdx.x & 255) < 2) found[threadIdx.x & 1] = 0;
      lds_barrier();
#pragma unroll 1
      for (int i = threadIdx.x & 255; i < kStep * 16 && live; i += 256) {
        const int r = i >> 4, key = t * kStep + r;
        if (key < see_all) continue;
        u32x4* p = reinterpret_cast<u32x4*>(buf + kV + r * 256 + (((i & 15) ^ swz_v(r)) << 4));
        u32x4 x = {0u, 0u, 0u, 0u};
        if (key < see_any) {
          x = *p;
          bool bad = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const bool lo = (x[w] & 0x7f80u) == 0x7f80u, hi = (x[w] & 0x7f800000u) == 0x7f800000u;
            if (lo) x[w] &= 0xffff0000u;
            if (hi) x[w] &= 0x0000ffffu;
            bad = bad || lo || hi;
          }
          if (bad) atomicOr(&found[r >> 5], 1u << (r & 31));
        }
        *p = x;
      }
      lds_barrier();
      odd = (unsigned long long)(unsigned)uniform(found[1]) << 32 | (unsigned)uniform(found[0]);
    }

    if (!live) continue;
    // ---- the first values are read under the softmax; 32 keys at a time: the lane's keys are 4g .. 4g + 3 of both
    // 16-key blocks; lane 4j + i reads elements 4i of key row 4g + j
    const int row = 4 * g + (r16 >> 2);
    const uint32_t at = (uint32_t)(buffer + kV) + row * 256 + (lane & 1) * 8 +
                        ((((lane >> 1) & 1) ^ swz_v(row)) << 4);
    const auto frag = [&](int i) __attribute__((always_inline)) {  // i = (half, block)
      const uint8_t* x = lds + (at ^ (i % CT << 5)) + i / CT * 32 * 256;
      const u32x2 v0 = lds_tr16(x), v1 = lds_tr16(x + 16 * 256);
      return u32x4{v0[0], v0[1], v1[0], v1[1]};
    };
    u32x4 ring[kAheadV];
#pragma unroll
    for (int i = 0; i < kAheadV; ++i) ring[i] = frag(i);
    __builtin_amdgcn_sched_barrier(0);
    // ---- softmax of the lane's queries
    float top[QF];
    bool move = false;
#pragma unroll
    for (int f = 0; f < QF; ++f) {
      float x = sc[0][f][0];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x = fmaxf(x, sc[k][f][i]);
      top[f] = rows_max(x) * a.scale_log2;
      move = move || top[f] > m[f] + kLazy;
    }
    if (__any(move)) {
#pragma unroll
      for (int f = 0; f < QF; ++f) {
        const float to = fmaxf(m[f], top[f]);
        const float by = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[f] - to);
        m[f] = to;
        l[f] *= by;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][f] *= by;
      }
    }
    u32x4 p[KT / 2][QF];
#pragma unroll
    for (int f = 0; f < QF; ++f) {
      const float base = m[f] == -INFINITY ? 0.f : m[f];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(sc[k][f][i], a.scale_log2, -base));
          l[f] += e[i];
        }
        p[k >> 1][f][2 * (k & 1)] = pack_bf16x2(e[0], e[1]);
        p[k >> 1][f][2 * (k & 1) + 1] = pack_bf16x2(e[2], e[3]);
      }
    }

    // ---- O^T += V^T P^T
    static_for<0, KT / 2 * CT>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, h = i / CT, c = i % CT;
      const u32x4 v = ring[i % kAheadV];
      if constexpr (i + kAheadV < KT / 2 * CT) ring[i % kAheadV] = frag(i + kAheadV);
#pragma unroll
      for (int f = 0; f < QF; ++f) o[c][f] = mfma_bf16_16x16x32(v, p[h][f], o[c][f]);
      if constexpr (i % kFence == kFence - 1) __builtin_amdgcn_sched_barrier(0);
    });
    while (odd != 0) {  // Inf and NaN to the tokens that see them
      const int r = __ffsll((long long)odd) - 1, key = t * kStep + r;
      odd &= odd - 1;
      const uint16_t* x = reinterpret_cast<const uint16_t*>(vv) + (long long)key * a.v_s + 4 * g;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(x + c * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = (i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
          const float add = (bits & 0x7f800000u) == 0x7f800000u ? __uint_as_float(bits) : 0.f;
#pragma unroll
          for (int f = 0; f < QF; ++f) o[c][f][i] += key < sees[f] ? add : 0.f;
        }
      }
    }
  }

#pragma unroll
  for (int f = 0; f < QF; ++f) {
    l[f] += __shfl_xor(l[f], 16, 64);
    l[f] += __shfl_xor(l[f], 32, 64);
  }
  const auto put = [&](int f, float top, float sum, auto&& value) __attribute__((always_inline)) {
    const int r = row0 + (wave * QF + f) * 16 + r16;
    if (r > row_last) return;
    const long long at = (long long)(q0 + r) * a.H + head;
    if constexpr (SPLIT) {
      const long long to = (long long)part * a.T * a.H + at;
#pragma unroll
      for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4*>(a.part() + to * kValue + c * 16 + 4 * g) = value(c);
      if (g == 0) a.ml[to] = make_float2(top, sum);
      return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* out = a.out + at * kValue + 4 * g;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const f32x4 x = value(c) * inv;
      *reinterpret_cast<u32x2*>(out + c * 16) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    }
    if (a.lse != nullptr && g == 0) a.lse[at] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  };
  if constexpr (TEAMS == 1) {
#pragma unroll
    for (int f = 0; f < QF; ++f) put(f, m[f], l[f], [&](int c) { return o[c][f]; });
  } else {
    // Each team finishes one of the two fragments of its queries.
    lds_barrier();  // the last steps have been read
    const auto finish = [&](auto kc) __attribute__((always_inline)) {
      constexpr int keep = decltype(kc)::value, send = 1 - keep;
      f32x4* to = reinterpret_cast<f32x4*>(lds) + (send * 4 + wave) * CT * 64 + lane;
      float2* stat = reinterpret_cast<float2*>(lds + TEAMS * 4 * CT * 64 * sizeof(f32x4));
#pragma unroll
      for (int c = 0; c < CT; ++c) to[c * 64] = o[c][send];
      stat[(send * 4 + wave) * 64 + lane] = make_float2(m[send], l[send]);
      lds_barrier();
      const f32x4* from = reinterpret_cast<const f32x4*>(lds) + (keep * 4 + wave) * CT * 64 + lane;
      const float2 other = stat[(keep * 4 + wave) * 64 + lane];
      const float top = fmaxf(m[keep], other.x), base = top == -INFINITY ? 0.f : top;
      const float mine = __builtin_amdgcn_exp2f(m[keep] - base), theirs = __builtin_amdgcn_exp2f(other.x - base);
      // l may be NaN where the maximum is -inf (a NaN that is the team's only key), and so is the sum then
      const float sum = (l[keep] != 0.f ? l[keep] * mine : 0.f) + (other.y != 0.f ? other.y * theirs : 0.f);
      put(keep, top, sum, [&](int c) { return o[c][keep] * mine + from[c * 64] * theirs; });
    };
    if (team == 0) finish(IntC<0>{});
    else finish(IntC<1>{});
  }
}

// Joins the parts of a row, 32 lanes of 4 columns each; rows behind the last sequence
// have none.
__global__ __launch_bounds__(256) void expanded_join_kernel(Args a) {
  const long long rows = (long long)a.T * a.H, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row < (long long)max(a.cu_q[0], 0) * a.H || row >= (long long)min(a.cu_q[a.B], a.T) * a.H) return;
  const float* part = a.part() + row * kValue + (threadIdx.x & 31) * 4;
  float2 ml[kMaxParts];
  f32x4 x[kMaxParts];
#pragma unroll
  for (int i = 0; i < kMaxParts; ++i) {
    ml[i] = make_float2(-INFINITY, 0.f);
    x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (i < a.parts) {
      ml[i] = a.ml[i * rows + row];
      x[i] = *reinterpret_cast<const f32x4*>(part + i * rows * kValue);
    }
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxParts; ++i) top = fmaxf(top, ml[i].x);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxParts; ++i) {
    const float by = __builtin_amdgcn_exp2f(ml[i].x - base);
    acc += x[i] * by;
    sum += ml[i].y != 0.f ? ml[i].y * by : 0.f;  // NaN where a NaN is a part's only key
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  acc *= inv;
  *reinterpret_cast<u32x2*>(a.out + row * kValue + (threadIdx.x & 31) * 4) =
      u32x2{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
  if (a.lse != nullptr && (threadIdx.x & 31) == 0)
    a.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Tiles that B sequences with T tokens can have.
long long tiles_of(int B, int T) { return std::min<long long>(T, (T + (kTokens - 1LL) * B) / kTokens); }

// Parts of a tile's keys: as many as there are CUs for, of kPartSteps steps or more by the
// keys that a token sees on average, as though all were causal.  One part / as here, us: 8
// heads, 100 tokens of 8192 keys 148 / 26.7 (16 parts), 1024 of 8192 148 / 59.9 (4), 2048
// of 8192 149 / 96.8 (2), 2048 of 2048 45.4 / 39.0 (2).  Against it: 16 heads, 1024 of
// 1024, 28.6 in one and 31.1 in two parts of 4 steps, whose partials cost more than
// they gain; 8 heads, 2048 of 8192, 128 in parts for four times as many CUs.
int parts_of(int B, int T, int S, int H) {
  const long long wide = kCus / (tiles_of(B, T) * H), deep = (S - T / 2) / B / (kStep * kPartSteps);
  return (int)std::max(1LL, std::min({wide, deep, (long long)kMaxParts}));
}

// One team or two, by the time that each is expected to take: either the longest tile
// decides (1.6 us a step in one team that has a CU to itself, half of 2.5 in two), or the
// sum over the card (2.45 us for two steps of a CU's two work-groups, 2.5 for two teams'
// and about 3 us for each of their tiles' start and join, which nothing covers).  One / two,
// causal, us: 16 heads, one prompt of 2048 56.2 / 47.1, of 4096 109 / 97.6, 4096 after 4096
// others 240 / 254, two of 2048 62.1 / 60.3, five of 1024 50.9 / 64.4, eight 74.1 / 102;
// 128 heads of 512 27.2 / 34.4.  The longest prompt is taken to be as long as the mean: a ragged
// batch's longest tile may count for more.
bool one_team(int B, int T, int S, long long groups) {
  const float longest = (float)S / B / kStep, mean = fmaxf((float)S - 0.5f * T, 0.f) / B / kStep;
  const float all = (float)groups * mean / (2 * kCus);
  return fmaxf(1.6f * longest, 2.45f * all) < fmaxf(1.25f * longest, 2.5f * all + 3.f * (float)groups / kCus);
}

template <int TEAMS, bool SPLIT>
hipError_t launch(const Args& a, long long groups, hipStream_t stream) {
  constexpr int lds = TEAMS * 2 * kBuf;
  if (const hipError_t e = set_lds_limit_once<expanded_attention_kernel<TEAMS, SPLIT>>(lds); e != hipSuccess) return e;
  hipLaunchKernelGGL((expanded_attention_kernel<TEAMS, SPLIT>), dim3((unsigned)groups), dim3(256 * TEAMS), lds, stream,
                     a);
  return hipGetLastError();
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" size_t ferret_latent_attention_expanded_workspace(int B, int T, int S, int H) {
  if (B < 1 || T < 1 || S < 1 || H < 1 || H > 1024) return 0;
  const int parts = parts_of(B, T, S, H);
  const size_t rows = (size_t)parts * T * H;
  return parts > 1 ? stat_bytes(rows) + rows * kValue * sizeof(float) : 0;
}

extern "C" int ferret_latent_attention_expanded(const void* q_nope, long long qn_token, long long qn_head,
                                                const void* q_rotary, long long qr_token, long long qr_head,
                                                const void* k_nope, long long kn_key, long long kn_head,
                                                const void* k_rotary, long long kr_key, const void* v, long long v_key,
                                                long long v_head, const int32_t* cu_q, const int32_t* cu_k, int B,
                                                int T, int S, int H, float scale, int causal, void* out, float* lse,
                                                void* ws, size_t ws_bytes, void* stream) {
  FERRET_REQUIRE(q_nope && q_rotary && k_nope && k_rotary && v && cu_q && cu_k && out, FERRET_ERR_NULL);
  FERRET_REQUIRE(B >= 1 && T >= 1 && S >= 1 && H >= 1 && H <= 1024, FERRET_ERR_SHAPE);
  FERRET_REQUIRE(S <= 1 << 30, FERRET_ERR_SHAPE);  // the search for a tile looks some steps past S
  FERRET_REQUIRE(scale > 0.f && scale < 1e30f, FERRET_ERR_SHAPE);
  for (const long long stride : {qn_token, qn_head, qr_token, qr_head, kn_key, kn_head, kr_key, v_key, v_head}) {
    FERRET_REQUIRE(stride >= 0 && stride < (1LL << 24), FERRET_ERR_SHAPE);  // 64 rows stay within 32 bits
    FERRET_REQUIRE(stride % 8 == 0, FERRET_ERR_ALIGN);
  }
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE(((bits(q_nope) | bits(q_rotary) | bits(k_nope) | bits(k_rotary) | bits(v) | bits(out)) & 15) == 0 &&
                     (bits(lse) & 3) == 0,
                 FERRET_ERR_ALIGN);
  const int parts = parts_of(B, T, S, H);
  const long long groups = tiles_of(B, T) * H * parts;
  FERRET_REQUIRE(groups < (1LL << 31), FERRET_ERR_SHAPE);
  const size_t need = ferret_latent_attention_expanded_workspace(B, T, S, H);
  FERRET_REQUIRE(parts == 1 || (ws != nullptr && (bits(ws) & 15) == 0 && ws_bytes >= need), FERRET_ERR_WORKSPACE);
  // In place is sound: a work-group writes the rows that it alone has read, or the join does.
  const bool over = in_place(out, q_nope, T, qn_token, H, qn_head, kNope);
  FERRET_REQUIRE(!clash({Range{out, (uint64_t)T * H * kValue * 2}, Range{lse, (uint64_t)T * H * 4},
                         Range{ws, need}},
                        {bf16_range(over ? nullptr : q_nope, T, qn_token, H, qn_head, kNope),
                         bf16_range(q_rotary, T, qr_token, H, qr_head, kRope),
                         bf16_range(k_nope, S, kn_key, H, kn_head, kNope), bf16_range(k_rotary, S, kr_key, 1, 0, kRope),
                         bf16_range(v, S, v_key, H, v_head, kValue), Range{cu_q, 4 * (B + 1ULL)},
                         Range{cu_k, 4 * (B + 1ULL)}}),
                 FERRET_ERR_SHAPE);
  Args a;
  a.qn = static_cast<const uint16_t*>(q_nope);
  a.qr = static_cast<const uint16_t*>(q_rotary);
  a.kn = static_cast<const uint16_t*>(k_nope);
  a.kr = static_cast<const uint16_t*>(k_rotary);
  a.v = static_cast<const uint16_t*>(v);
  a.qn_t = (int)qn_token;
  a.qn_h = (int)qn_head;
  a.qr_t = (int)qr_token;
  a.qr_h = (int)qr_head;
  a.kn_s = (int)kn_key;
  a.kn_h = (int)kn_head;
  a.kr_s = (int)kr_key;
  a.v_s = (int)v_key;
  a.v_h = (int)v_head;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.B = B;
  a.T = T;
  a.S = S;
  a.H = H;
  a.scale_log2 = scale * kLog2e;
  a.causal = causal != 0;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.parts = parts;
  a.ml = static_cast<float2*>(ws);
  const hipStream_t on = (hipStream_t)stream;
  if (parts > 1) {
    FERRET_HIP_CHECK((launch<2, true>(a, groups, on)));
    const long long rows = (long long)T * H;
    hipLaunchKernelGGL(expanded_join_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, on, a);
    return (int)hipGetLastError();
  }
  return (int)(one_team(B, T, S, groups) ? launch<1, false>(a, groups, on) : launch<2, false>(a, groups, on));
}
