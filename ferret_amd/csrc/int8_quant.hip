// bf16 rows to int8 codes with one fp32 scale per token, the activations of the
// int8 product:
//   a = max(max_k |x[m,k]|, 2^-100),  q[m,k] = RNE(127 x[m,k] / a),  scale[m] = a / 127
// The codes are those of the exact quotient, ties to even: t = u * (128 / a) of
// the exact u = 127/128 x is carried on by its exact remainder, t + (u - t a / 128) *
// (128 / a), which gives a half exactly where the quotient is one (it has 8 bits);
// elsewhere a half is 2^-18 or more away, over the error of the sum.  A row with an
// Inf or NaN gets zeros and the scale NaN, so that its products are NaN.
//
// One pass: a row stays in the registers of the WPR waves that own it, its largest
// value as a 15-bit pattern (unsigned maxima order Inf and NaN above all numbers).
// HBM-bound: 2 bytes read and 1 written per element.  8192 rows of 7168 take 29.0 us, 6.1
// TB/s; 32 rows of 4096 2.8 us in the kernel, the launch.
//
// As many waves per row as leave a lane two chunks: more loads of a lane wait longer for
// the first, fewer leave little to do between the two passes.  Us, 32 / 1000 / 8192 rows: K 4096,
// 8 x 1 2.9 / 4.5 / 22.7, 4 x 2 3.0 / 4.1 / 20.3, 2 x 4 3.5 / 4.1 / 19.2; K 7168, 16 x 1 3.1 / 7.3 / 38.6, 8 x 2
// 3.0 / 6.0 / 29.7, 4 x 4 3.5 / 6.6 / 32.5; K 2048, 4 x 1 2.8 / 3.5 / 13.3, 2 x 2 3.0 / 3.3 / 11.9, 1 x 4
// 3.2 / 3.9 / 12.7.
#include "common.hpp"
#include "ranges.hpp"

namespace ferret {
namespace {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

struct QuantArgs {
  const uint16_t* x;
  uint8_t* q;
  float* scale;
  long long x_stride;
  int M, K;
};

__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// WPR waves per row, CH chunks of 8 elements per lane: 64 * WPR * CH * 8 >= K.
template <int WPR, int CH>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void quant_int8_kernel(QuantArgs a) {
  constexpr int ROWS = WPR >= 4 ? 1 : 4 / WPR;  // rows per work-group
  constexpr int LANES = 64 * WPR;
  __shared__ uint32_t part[ROWS * WPR];
  const int row_in = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * ROWS + row_in;
  const bool live = row < a.M;
  const int chunks = a.K >> 3;
  u32x4 v[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = c * LANES + lane;
    v[c] = live && k < chunks ? ld_u32x4_stream(a.x + row * a.x_stride + (long long)k * 8) : u32x4{0u, 0u, 0u, 0u};
  }
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max_pair(top, v[c][i] & 0x7fff7fffu);
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  if constexpr (WPR > 1) {
    if ((lane & 63) == 0) part[row_in * WPR + (lane >> 6)] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, part[row_in * WPR + i]);
  }
  const bool bad = top >= 0x7f80u;
  const float amax = fmaxf(__uint_as_float(top << 16), 0x1p-100f);
  const float inv = 128.f / amax, unit = amax * 0x1p-7f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = c * LANES + lane;
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __uint_as_float(i & 1 ? v[c][i >> 1] & 0xffff0000u : v[c][i >> 1] << 16);
      const float u = x * 0.9921875f, t = u * inv;
      const float exact = fmaf(fmaf(-t, unit, u), inv, t);
      code[i] = __float_as_uint(exact + 12582912.f);  // 1.5 * 2^23: the low byte is the rounded code
    }
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __builtin_amdgcn_perm(code[4 * h + 1], code[4 * h], 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(code[4 * h + 3], code[4 * h + 2], 0x04000c0cu);
      w[h] = bad ? 0u : lo | hi;
    }
    if (live && k < chunks) *reinterpret_cast<u32x2*>(a.q + row * a.K + (long long)k * 8) = w;
  }
  if (live && lane == 0) a.scale[row] = bad ? __uint_as_float(0x7fc00000u) : amax / 127.f;
}

template <int WPR, int CH>
int launch(const QuantArgs& a, hipStream_t st) {
  constexpr int ROWS = WPR >= 4 ? 1 : 4 / WPR;
  constexpr int THREADS = WPR > 4 ? 64 * WPR : 256;
  const long long grid = ((long long)a.M + ROWS - 1) / ROWS;
  hipLaunchKernelGGL((quant_int8_kernel<WPR, CH>), dim3((unsigned)grid), dim3(THREADS), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" int ferret_quant_act_int8(const void* x, long long x_stride, int M, int K, void* q, float* scale,
                                     void* stream) {
  FERRET_REQUIRE(x != nullptr && q != nullptr && scale != nullptr, FERRET_ERR_NULL);
  FERRET_REQUIRE(M >= 1 && M < (1 << 22) && K >= 16 && K <= 32768 && K % 16 == 0, FERRET_ERR_SHAPE);  // 2^32 threads
  FERRET_REQUIRE(M == 1 || (x_stride >= K && x_stride < (1LL << 40)), FERRET_ERR_SHAPE);
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE((bits(x) & 15) == 0 && (bits(q) & 15) == 0 && (bits(scale) & 3) == 0 && (M == 1 || x_stride % 8 == 0),
                 FERRET_ERR_ALIGN);
  FERRET_REQUIRE(!clash({Range{q, (uint64_t)M * K}, Range{scale, (uint64_t)M * 4}},
                        {bf16_range(x, M, M == 1 ? 0 : x_stride, 1, 0, K)}),
                 FERRET_ERR_SHAPE);
  const QuantArgs a{static_cast<const uint16_t*>(x), static_cast<uint8_t*>(q), scale, x_stride, M, K};
  const hipStream_t st = (hipStream_t)stream;
  const int chunks = K / 8;
  if (chunks <= 64) return launch<1, 1>(a, st);
  if (chunks <= 128) return launch<1, 2>(a, st);
  if (chunks <= 256) return launch<2, 2>(a, st);
  if (chunks <= 512) return launch<4, 2>(a, st);
  if (chunks <= 1024) return launch<8, 2>(a, st);
  if (chunks <= 2048) return launch<16, 2>(a, st);
  return launch<16, 4>(a, st);
}
