// Root-mean-square norm of bf16 rows with the residual's addition, the step
// before every projection:
//   s = x + r                      (fp32; stored as bf16 where r is given)
//   y = s * rsqrt(mean(s^2) + eps) * w
// and y as bf16, or as the e4m3 codes and 1x128 scales that the FP8 products
// take (the rule of quant_act_e4m3 on the fp32 y):
//   a = max(max_{block} |y|, 1e-4),  q = e4m3_RNE(y * (448 / a)),  scale = a / 448
// The norm is taken of the fp32 sum, not of its bf16 copy: one rounding per
// result.  Sums are fp32, in an order that K alone fixes.
//
// One pass: a row stays in the registers of the WPR waves that own it (CH
// 16-byte chunks per lane), so it is read once, and a row may be written in
// place: every lane's loads have returned before its row's sum is known.
// HBM-bound: 2 bytes read per element (4 with the residual) and 1 to 4 written.  8192
// rows of 7168 with residual and codes: 71 us, 5.8 TB/s; 64 rows of 512: 2.3 us in a
// replayed graph, 5.0 called from Python, the launch.
#include "common.hpp"
#include "ranges.hpp"

namespace ferret {

// Sum over the 64 lanes of a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Maximum over aligned groups of 16 lanes (one DPP row), in every lane.
__device__ __forceinline__ float row16_max(float v) {
#define FERRET_ROR_MAX(n)                                                                                    \
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 | (n), 0xf, 0xf, true)))
  FERRET_ROR_MAX(8);
  FERRET_ROR_MAX(4);
  FERRET_ROR_MAX(2);
  FERRET_ROR_MAX(1);
#undef FERRET_ROR_MAX
  return v;
}

struct NormArgs {
  const uint16_t* x;
  const uint16_t* r;
  const uint16_t* w;
  uint16_t* r_out;
  uint16_t* y;    // bf16 result
  uint8_t* q;     // or e4m3 codes
  float* scale;   // and their scales
  long long x_stride, r_stride;
  float eps;
  int M, K;
};

// WPR waves per row, CH chunks of 8 elements per lane: 64 * WPR * CH * 8 >= K.
template <int WPR, int CH, bool RES, bool F8>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void rms_norm_kernel(NormArgs a) {
  constexpr int ROWS = WPR >= 4 ? 1 : 4 / WPR;  // rows per work-group
  constexpr int LANES = 64 * WPR;
  __shared__ float part[ROWS * WPR];
  const int row_in = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * ROWS + row_in;
  const bool live = row < a.M;
  const int chunks = a.K >> 3;
  u32x4 vx[CH], vr[CH], vw[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = c * LANES + lane;
    const bool in = live && k < chunks;
    vx[c] = in ? ld_u32x4_stream(a.x + row * a.x_stride + (long long)k * 8) : u32x4{0u, 0u, 0u, 0u};
    if constexpr (RES)
      vr[c] = in ? ld_u32x4_stream(a.r + row * a.r_stride + (long long)k * 8) : u32x4{0u, 0u, 0u, 0u};
    vw[c] = k < chunks ? ld_u32x4(a.w + (long long)k * 8) : u32x4{0u, 0u, 0u, 0u};
  }
  float s[CH][8];
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[c][2 * i] = __uint_as_float(vx[c][i] << 16);
      s[c][2 * i + 1] = __uint_as_float(vx[c][i] & 0xffff0000u);
      if constexpr (RES) {
        s[c][2 * i] += __uint_as_float(vr[c][i] << 16);
        s[c][2 * i + 1] += __uint_as_float(vr[c][i] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(s[c][i], s[c][i], sq);
  }
  sq = wave_sum(sq);
  if constexpr (WPR > 1) {
    if ((lane & 63) == 0) part[row_in * WPR + (lane >> 6)] = sq;
    __syncthreads();
    sq = part[row_in * WPR];
#pragma unroll
    for (int i = 1; i < WPR; ++i) sq += part[row_in * WPR + i];
  }
  const float rstd = rsqrtf(sq / (float)a.K + a.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = c * LANES + lane;
    const bool in = live && k < chunks;
    if constexpr (RES) {
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(s[c][2 * i], s[c][2 * i + 1]);
      if (in) *reinterpret_cast<u32x4*>(a.r_out + row * a.K + (long long)k * 8) = o;
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = s[c][2 * i] * rstd * __uint_as_float(vw[c][i] << 16);
      y[2 * i + 1] = s[c][2 * i + 1] * rstd * __uint_as_float(vw[c][i] & 0xffff0000u);
    }
    if constexpr (F8) {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
      amax = fmaxf(row16_max(amax), 1e-4f);  // a 128-element block is one aligned group of 16 lanes
      const float mult = 448.0f / amax;
      uint32_t lo = 0, hi = 0;
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * mult, y[1] * mult, lo, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * mult, y[3] * mult, lo, true);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * mult, y[5] * mult, hi, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * mult, y[7] * mult, hi, true);
      if (in) {
        *reinterpret_cast<u32x2*>(a.q + row * a.K + (long long)k * 8) = u32x2{lo, hi};
        if ((k & 15) == 0) a.scale[row * (a.K >> 7) + (k >> 4)] = amax / 448.0f;
      }
    } else {
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
      if (in) *reinterpret_cast<u32x4*>(a.y + row * a.K + (long long)k * 8) = o;
    }
  }
}

template <int WPR, int CH, bool RES, bool F8>
static int launch_norm(const NormArgs& a, hipStream_t st) {
  constexpr int ROWS = WPR >= 4 ? 1 : 4 / WPR;
  constexpr int THREADS = WPR > 4 ? 64 * WPR : 256;
  const long long grid = ((long long)a.M + ROWS - 1) / ROWS;
  hipLaunchKernelGGL((rms_norm_kernel<WPR, CH, RES, F8>), dim3((unsigned)grid), dim3(THREADS), 0, st, a);
  return (int)hipGetLastError();
}

// Waves per row by the chunks of a row.  One up to 192 chunks, four rows per work-group
// (8192 rows, codes out, us: K = 1024 8.0 against 10.6 with four waves, 1536 9.2 against
// 10.4 with two and 12.5 with four), two up to 256 (2048: 11.4 against 13.3 with four),
// eight up to 2048 (4096 and the residual 40.8 against 41.3 with four, 7168 70.0 against
// 71.5 with four and 74.8 with sixteen), and sixteen for the rows that those do not hold.
template <bool RES, bool F8>
static int pick_norm(const NormArgs& a, hipStream_t st) {
  const int chunks = a.K / 8;
  if (chunks <= 64) return launch_norm<1, 1, RES, F8>(a, st);
  if (chunks <= 128) return launch_norm<1, 2, RES, F8>(a, st);
  if (chunks <= 192) return launch_norm<1, 3, RES, F8>(a, st);
  if (chunks <= 256) return launch_norm<2, 2, RES, F8>(a, st);
  if (chunks <= 512) return launch_norm<8, 1, RES, F8>(a, st);
  if (chunks <= 1024) return launch_norm<8, 2, RES, F8>(a, st);
  if (chunks <= 2048) return launch_norm<8, 4, RES, F8>(a, st);
  return launch_norm<16, 4, RES, F8>(a, st);
}

static bool overlap(const void* a, long long a_bytes, const void* b, long long b_bytes) {
  return overlap(Range{a, (uint64_t)a_bytes}, Range{b, (uint64_t)b_bytes});
}

// Rows of `out` (K elements of `size` bytes, packed) over rows of `in`: only
// the very same rows may be written in place.
static bool clash(const void* out, int size, const void* in, long long in_stride, long long M, long long K) {
  if (in == nullptr || out == nullptr) return false;
  if (size == 2 && out == in && (in_stride == K || M == 1)) return false;
  return overlap(out, M * K * size, in, ((M - 1) * in_stride + K) * 2);
}

static int check_norm(const NormArgs& a, const void* y, int size) {
  FERRET_REQUIRE(a.x != nullptr && a.w != nullptr && y != nullptr, FERRET_ERR_NULL);
  FERRET_REQUIRE((a.r == nullptr) == (a.r_out == nullptr), FERRET_ERR_NULL);
  FERRET_REQUIRE(a.M >= 1 && a.K >= 8 && a.K <= 32768 && a.K % (size == 1 ? 128 : 8) == 0, FERRET_ERR_SHAPE);
  FERRET_REQUIRE(a.eps >= 0.f && a.eps < 1e30f, FERRET_ERR_SHAPE);
  FERRET_REQUIRE(a.M == 1 || (a.x_stride >= a.K && (a.r == nullptr || a.r_stride >= a.K)), FERRET_ERR_SHAPE);
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE(((bits(a.x) | bits(a.r) | bits(a.w) | bits(a.r_out)) & 15) == 0 &&
                     (bits(y) & (size == 1 ? 7 : 15)) == 0 && (bits(a.scale) & 3) == 0,
                 FERRET_ERR_ALIGN);
  FERRET_REQUIRE(a.M == 1 || (a.x_stride % 8 == 0 && (a.r == nullptr || a.r_stride % 8 == 0)), FERRET_ERR_ALIGN);
  const long long M = a.M, K = a.K, blocks = a.scale != nullptr ? M * (K / 128) * 4 : 0;
  FERRET_REQUIRE(!clash(y, size, a.x, a.x_stride, M, K) && !clash(y, size, a.r, a.r_stride, M, K) &&
                     !clash(a.r_out, 2, a.x, a.x_stride, M, K) && !clash(a.r_out, 2, a.r, a.r_stride, M, K) &&
                     !(a.r_out != nullptr && overlap(y, M * K * size, a.r_out, M * K * 2)) &&
                     !overlap(y, M * K * size, a.w, K * 2) &&
                     !(a.r_out != nullptr && overlap(a.r_out, M * K * 2, a.w, K * 2)),
                 FERRET_ERR_SHAPE);
  if (blocks != 0)
    FERRET_REQUIRE(!overlap(a.scale, blocks, y, M * K) && !overlap(a.scale, blocks, a.w, K * 2) &&
                       !overlap(a.scale, blocks, a.x, ((M - 1) * a.x_stride + K) * 2) &&
                       !(a.r != nullptr && (overlap(a.scale, blocks, a.r, ((M - 1) * a.r_stride + K) * 2) ||
                                            overlap(a.scale, blocks, a.r_out, M * K * 2))),
                   FERRET_ERR_SHAPE);
  return FERRET_OK;
}

}  // namespace ferret

using namespace ferret;

extern "C" int ferret_rms_norm(const void* x, long long x_stride, const void* residual, long long residual_stride,
                               const void* w, float eps, int M, int K, void* y, void* residual_out, void* stream) {
  const NormArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                   static_cast<const uint16_t*>(w), static_cast<uint16_t*>(residual_out), static_cast<uint16_t*>(y),
                   nullptr, nullptr, x_stride, residual_stride, eps, M, K};
  const int rc = check_norm(a, y, 2);
  if (rc != FERRET_OK) return rc;
  return residual != nullptr ? pick_norm<true, false>(a, (hipStream_t)stream)
                             : pick_norm<false, false>(a, (hipStream_t)stream);
}

extern "C" int ferret_rms_norm_e4m3(const void* x, long long x_stride, const void* residual,
                                    long long residual_stride, const void* w, float eps, int M, int K, void* q,
                                    float* scale, void* residual_out, void* stream) {
  const NormArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                   static_cast<const uint16_t*>(w), static_cast<uint16_t*>(residual_out), nullptr,
                   static_cast<uint8_t*>(q), scale, x_stride, residual_stride, eps, M, K};
  FERRET_REQUIRE(scale != nullptr, FERRET_ERR_NULL);
  const int rc = check_norm(a, q, 1);
  if (rc != FERRET_OK) return rc;
  return residual != nullptr ? pick_norm<true, true>(a, (hipStream_t)stream)
                             : pick_norm<false, true>(a, (hipStream_t)stream);
}
