// Latent attention in its expanded form: ragged prompts over per-head keys and values
// (128 + 64 and 128 wide), the 64 rotary key values shared by all heads:
//   s_ij = scale * (qn_i . kn_j + qr_i . kr_j),   o_i = sum_j softmax_j(s_ij) v_j
// for one head; token i of n new ones sees the keys j <= len - n + i of its sequence
// (causal) or all len.  A token that sees none gives zeros and lse -inf.
//
// A work-group takes 128 tokens of one head, 32 per wave, and walks the keys in steps
// of 64, which come into LDS by asynchronous loads, one step ahead.  S^T = K Q^T has
// the keys as MFMA rows: a lane holds the scores of one query and, per block, four
// consecutive keys, which is the operand that O^T = V^T P^T needs (the order of the
// keys within the contraction is free as long as V^T follows it), so P never leaves
// its registers.  V^T comes from row-major V by transposing LDS reads.  80 KB of LDS
// and half the registers leave room for two work-groups per CU: one's softmax runs
// under the other's products.  Tiles of a sequence go longest first, and a head's
// tiles to one XCD where the number of heads is a multiple of 8 (keys from its L2).
//
// MFMA-bound: 2 * (192 + 128) operations per query, visible key and head.  S, m, l and
// O are fp32; P is rounded to bf16 (half an ulp, 2^-9), l sums the unrounded terms.
#include "attention.hpp"

#include <initializer_list>

namespace ferret {
namespace {

constexpr int kNope = 128, kRope = 64, kValue = 128;
constexpr int kStep = 64;                              // keys per step
constexpr int kTokens = 128;                           // per work-group
constexpr int kKn = 0, kKr = kStep * kNope * 2;        // a buffer: keys, rotary keys, values
constexpr int kV = kKr + kStep * kRope * 2, kBuf = kV + kStep * kValue * 2;
constexpr int kLdsBytes = 2 * kBuf;
static_assert(2 * kLdsBytes <= 160 * 1024, "two work-groups per CU");

struct Args {
  const uint16_t *qn, *qr, *kn, *kr, *v;
  int qn_t, qn_h, qr_t, qr_h, kn_s, kn_h, kr_s, v_s, v_h;  // strides in elements
  const int32_t *cu_q, *cu_k;
  int B, T, S, H;
  float scale_log2;
  int causal;
  uint16_t* out;  // [T, H, 128]
  float* lse;     // [T, H] or null
};

// The swizzles: 16-byte chunk c of row r stands at c ^ swizzle(r).  Rows of 256
// bytes (a whole turn of the banks) and of 128.
__device__ __forceinline__ int swz_kn(int r) { return r & 15; }
__device__ __forceinline__ int swz_kr(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz_v(int r) { return 2 * (r & 7); }

__global__ __launch_bounds__(256, 2) void expanded_attention_kernel(Args a) {
  constexpr int QF = 2, KT = kStep / 16, CT = kValue / 16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.H;

  // ---- the tile: every wave finds it by itself
  int b = -1, tile = 0, left = blockIdx.x / a.H;
  for (int base = 0; base < a.B; base += 64) {
    int tiles = 0;
    if (base + lane < a.B) {
      const int q0 = min(max(a.cu_q[base + lane], 0), a.T), q1 = min(max(a.cu_q[base + lane + 1], q0), a.T);
      tiles = (q1 - q0 + kTokens - 1) / kTokens;
    }
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
  const int last = (min(see_any, len) + kStep - 1) / kStep;

  // ---- steps into LDS: this wave's 16 rows of each array (4, 8 and 4 rows per load)
  const uint8_t* kn = reinterpret_cast<const uint8_t*>(a.kn + (long long)k0 * a.kn_s + (long long)head * a.kn_h);
  const uint8_t* kr = reinterpret_cast<const uint8_t*>(a.kr + (long long)k0 * a.kr_s);
  const uint8_t* vv = reinterpret_cast<const uint8_t*>(a.v + (long long)k0 * a.v_s + (long long)head * a.v_h);
  const auto issue = [&](int t) {
    const uint32_t buf = uniform(lds_address(lds) + (t & 1) * kBuf);
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
  if (last > 0) issue(0);

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

  for (int t = 0; t < last; ++t) {
    wait_vmcnt<0>();
    lds_barrier();  // the step has landed for every wave, and the other buffer has been read
    if (t + 1 < last) issue(t + 1);
    __builtin_amdgcn_sched_barrier(0);
    uint8_t* buf = lds + (t & 1) * kBuf;

    // ---- S^T: 16 keys x 16 queries per block
    f32x4 sc[KT][QF];
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int f = 0; f < QF; ++f) sc[k][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    {
      const uint8_t* nope = buf + kKn + r16 * 256;
      const uint8_t* rope = buf + kKr + r16 * 128;
      const int zn = (g ^ (r16 & 3)) << 4, zr = (g ^ (swz_kr(r16) & 3)) << 4;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 c = ld_u32x4(nope + k * 16 * 256 + (zn | ((j ^ (r16 >> 2)) << 6)));
#pragma unroll
          for (int f = 0; f < QF; ++f) sc[k][f] = mfma_bf16_16x16x32(c, qf[f][j], sc[k][f]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const u32x4 c = ld_u32x4(rope + k * 16 * 128 + (zr | ((j ^ (swz_kr(r16) >> 2)) << 6)));
#pragma unroll
          for (int f = 0; f < QF; ++f) sc[k][f] = mfma_bf16_16x16x32(c, qf[f][4 + j], sc[k][f]);
        }
      }
    }

    // ---- masks: only where the step passes what some token of the tile sees
    unsigned long long odd = 0;  // rows with Inf or NaN among the values that not all tokens see
    if ((t + 1) * kStep > see_all) {
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
      if (threadIdx.x < 2) found[threadIdx.x] = 0;
      lds_barrier();
#pragma unroll 1
      for (int i = threadIdx.x; i < kStep * 16; i += 256) {
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
      x = fmaxf(x, __shfl_xor(x, 16, 64));
      top[f] = fmaxf(x, __shfl_xor(x, 32, 64)) * a.scale_log2;
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

    // ---- O^T += V^T P^T, 32 keys at a time: the lane's keys are 4g .. 4g + 3 of both
    // 16-key blocks; lane 4j + i reads elements 4i of key row 4g + j
    {
      const int row = 4 * g + (r16 >> 2);
      const uint32_t at = (uint32_t)((t & 1) * kBuf + kV) + row * 256 + (lane & 1) * 8 +
                          ((((lane >> 1) & 1) ^ swz_v(row)) << 4);
#pragma unroll
      for (int h = 0; h < KT / 2; ++h)
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const uint8_t* x = lds + (at ^ (c << 5)) + h * 32 * 256;
          const u32x2 v0 = lds_tr16(x), v1 = lds_tr16(x + 16 * 256);
          const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
          for (int f = 0; f < QF; ++f) o[c][f] = mfma_bf16_16x16x32(v, p[h][f], o[c][f]);
        }
    }
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
    float sum = l[f];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    const int r = row0 + (wave * QF + f) * 16 + r16;
    if (r > row_last) continue;
    const long long at = (long long)(q0 + r) * a.H + head;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* to = a.out + at * kValue + 4 * g;
#pragma unroll
    for (int c = 0; c < CT; ++c)
      *reinterpret_cast<u32x2*>(to + c * 16) =
          u32x2{pack_bf16x2(o[c][f][0] * inv, o[c][f][1] * inv), pack_bf16x2(o[c][f][2] * inv, o[c][f][3] * inv)};
    if (a.lse != nullptr && g == 0) a.lse[at] = sum == 0.f ? -INFINITY : (m[f] + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" int ferret_latent_attention_expanded(const void* q_nope, long long qn_token, long long qn_head,
                                                const void* q_rotary, long long qr_token, long long qr_head,
                                                const void* k_nope, long long kn_key, long long kn_head,
                                                const void* k_rotary, long long kr_key, const void* v, long long v_key,
                                                long long v_head, const int32_t* cu_q, const int32_t* cu_k, int B,
                                                int T, int S, int H, float scale, int causal, void* out, float* lse,
                                                void* stream) {
  FERRET_REQUIRE(q_nope && q_rotary && k_nope && k_rotary && v && cu_q && cu_k && out, FERRET_ERR_NULL);
  FERRET_REQUIRE(B >= 1 && T >= 1 && S >= 1 && H >= 1 && H <= 1024, FERRET_ERR_SHAPE);
  FERRET_REQUIRE(scale > 0.f && scale < 1e30f, FERRET_ERR_SHAPE);
  for (const long long stride : {qn_token, qn_head, qr_token, qr_head, kn_key, kn_head, kr_key, v_key, v_head}) {
    FERRET_REQUIRE(stride >= 0 && stride < (1LL << 24), FERRET_ERR_SHAPE);  // 64 rows stay within 32 bits
    FERRET_REQUIRE(stride % 8 == 0, FERRET_ERR_ALIGN);
  }
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE(((bits(q_nope) | bits(q_rotary) | bits(k_nope) | bits(k_rotary) | bits(v) | bits(out)) & 15) == 0 &&
                     (bits(lse) & 3) == 0,
                 FERRET_ERR_ALIGN);
  const long long tiles = T / kTokens + (B < T ? B : T);
  FERRET_REQUIRE(tiles * H < (1LL << 31), FERRET_ERR_SHAPE);
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
  FERRET_HIP_CHECK((set_lds_limit_once<expanded_attention_kernel>(kLdsBytes)));
  hipLaunchKernelGGL(expanded_attention_kernel, dim3((unsigned)(tiles * H)), dim3(256), kLdsBytes,
                     (hipStream_t)stream, a);
  return (int)hipGetLastError();
}
