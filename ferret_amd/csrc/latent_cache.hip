// Writing new tokens' latents and rotary keys into the paged cache, and reading
// the rows of a batch back (formats and page rules: latent.hpp).
//
// e4m3 write, per 128 latents of a token:  a = max |x| over the finite values,
//   e = ceil(log2(a / 448)),  byte = max(e + 127, 16),  code = e4m3_RNE(x * 2^-e)
// exactly: e comes from a's exponent and mantissa bits (448 = 1.75 * 2^8, so a
// block whose mantissa is past 1.75 needs the next power), and the product with a
// power of two does not round.  Inf and NaN become the NaN code.
//
// One wave per token: a lane holds 8 latents (16 lanes are a block), lanes 0 - 7
// the rotary values.  HBM-bound: 1152 bytes on one side and 644 (e4m3) or 1152 on
// the other; at decode sizes the launch and the two dependent loads (cu_q, page
// table) are all there is.  48000 rows read from e4m3: 22.7 us, 3.8 TB/s (two and four
// rows per wave, their loads in flight together: 23.3 and 30.5); in a replayed graph 64
// tokens written take 2.6 us and 9900 tokens 6.5, where their bytes take 3.6: a wave per
// token, whose look-ups (cu_q, the length, the page table) follow one another.
#include "latent.hpp"

namespace ferret {

__device__ __forceinline__ uint32_t row16_max_u32(uint32_t v) {
#define FERRET_ROR_UMAX(n)                                                                         \
  {                                                                                                \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 | (n), 0xf, 0xf, true); \
    v = v > o ? v : o;                                                                             \
  }
  FERRET_ROR_UMAX(8)
  FERRET_ROR_UMAX(4)
  FERRET_ROR_UMAX(2)
  FERRET_ROR_UMAX(1)
#undef FERRET_ROR_UMAX
  return v;
}

template <bool F8>
__global__ __launch_bounds__(256) void cache_write_kernel(const uint16_t* __restrict__ latent, long long ls,
                                                          const uint16_t* __restrict__ rotary, long long rs,
                                                          const int32_t* __restrict__ lens,
                                                          const int32_t* __restrict__ cu_q, int B, int T, Pages pages,
                                                          uint8_t* __restrict__ data, uint32_t* __restrict__ scales) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= T) return;  // whole waves
  const u32x4 v = ld_u32x4_stream(latent + t * ls + lane * 8);
  u32x4 rot = {0u, 0u, 0u, 0u};
  if (lane < 8) rot = ld_u32x4_stream(rotary + t * rs + lane * 8);
  const int b = sequence_of(cu_q, B, t);
  if (b >= B || t < cu_q[b]) return;
  const long long pos = (long long)lens[b] - cu_q[b + 1] + t;  // 32 bits would go round far below zero
  if (pos < 0 || pos > INT_MAX) return;
  const long long row = cache_row(pages, b, (int)pos);
  if (row < 0) return;
  if constexpr (!F8) {
    uint8_t* to = data + row * kRowBf16;
    *reinterpret_cast<u32x4*>(to + lane * 16) = v;
    if (lane < 8) *reinterpret_cast<u32x4*>(to + 2 * kLatent + lane * 16) = rot;
  } else {
    // |x| of the finite values as fp32 bits: they order as integers.
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = (v[i] << 16) & 0x7fffffffu, hi = v[i] & 0x7fff0000u;
      if (lo < 0x7f800000u && lo > amax) amax = lo;
      if (hi < 0x7f800000u && hi > amax) amax = hi;
    }
    amax = row16_max_u32(amax);
    int byte = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    byte = byte < kMinByte ? kMinByte : byte;
    const float mult = __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^(127 - byte)
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16) * mult;
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u) * mult;
    }
    uint32_t lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
    uint8_t* to = data + row * kRowE4m3;
    *reinterpret_cast<u32x2*>(to + lane * 8) = u32x2{lo, hi};
    if (lane < 8) *reinterpret_cast<u32x4*>(to + kLatent + lane * 16) = rot;
    const uint32_t word = (uint32_t)__builtin_amdgcn_readlane(byte, 0) |
                          (uint32_t)__builtin_amdgcn_readlane(byte, 16) << 8 |
                          (uint32_t)__builtin_amdgcn_readlane(byte, 32) << 16 |
                          (uint32_t)__builtin_amdgcn_readlane(byte, 48) << 24;
    if (lane == 0) scales[row] = word;
  }
}

template <bool F8>
__global__ __launch_bounds__(256) void cache_read_kernel(const uint8_t* __restrict__ data,
                                                         const uint32_t* __restrict__ scales,
                                                         const int32_t* __restrict__ cu_k, int B, int rows,
                                                         Pages pages, uint16_t* __restrict__ latent,
                                                         uint16_t* __restrict__ rotary) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= rows) return;  // whole waves
  const int b = sequence_of(cu_k, B, r);
  if (b >= B || r < cu_k[b]) return;
  const long long row = cache_row(pages, b, r - cu_k[b]);
  u32x4 o = {0u, 0u, 0u, 0u}, rot = {0u, 0u, 0u, 0u};
  if (row >= 0) {
    if constexpr (!F8) {
      const uint8_t* from = data + row * kRowBf16;
      o = ld_u32x4_stream(from + lane * 16);
      if (lane < 8) rot = ld_u32x4_stream(from + 2 * kLatent + lane * 16);
    } else {
      const uint8_t* from = data + row * kRowE4m3;
      const u32x2 c = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(from + lane * 8));
      if (lane < 8) rot = ld_u32x4_stream(from + kLatent + lane * 16);
      const uint32_t byte = (scales[row] >> ((lane >> 4) * 8)) & 255u;
      o = __builtin_bit_cast(u32x4, e4m3x8_to_bf16x8_scaled(c[0], c[1], __uint_as_float(byte << 23)));
    }
  }
  *reinterpret_cast<u32x4*>(latent + (long long)r * kLatent + lane * 8) = o;
  if (lane < 8) *reinterpret_cast<u32x4*>(rotary + (long long)r * kRotary + lane * 8) = rot;
}

static uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace ferret

using namespace ferret;

int ferret_check_pages(const int32_t* page_table, int B, int max_pages, int pages, int page_size) {
  FERRET_REQUIRE(page_table != nullptr, FERRET_ERR_NULL);
  FERRET_REQUIRE(B >= 1 && max_pages >= 1 && pages >= 1 && page_size >= 16 && page_size % 16 == 0, FERRET_ERR_SHAPE);
  FERRET_REQUIRE((long long)max_pages * page_size < (1LL << 31), FERRET_ERR_SHAPE);
  return FERRET_OK;
}

extern "C" int ferret_latent_cache_write(const void* latent, long long latent_stride, const void* rotary,
                                         long long rotary_stride, const int32_t* page_table, const int32_t* lens,
                                         const int32_t* cu_q, int B, int max_pages, int T, void* data, void* scales,
                                         int pages, int page_size, void* stream) {
  FERRET_REQUIRE(latent && rotary && lens && cu_q && data, FERRET_ERR_NULL);
  const int rc = ferret_check_pages(page_table, B, max_pages, pages, page_size);
  if (rc != FERRET_OK) return rc;
  FERRET_REQUIRE(T >= 1 && (T == 1 || (latent_stride >= kLatent && rotary_stride >= kRotary)), FERRET_ERR_SHAPE);
  FERRET_REQUIRE(((bits(latent) | bits(rotary) | bits(data)) & 15) == 0 && (bits(scales) & 3) == 0 &&
                     (T == 1 || (latent_stride % 8 == 0 && rotary_stride % 8 == 0)),
                 FERRET_ERR_ALIGN);
  FERRET_REQUIRE(!clash({data_range(data, scales, pages, page_size), scale_range(scales, pages, page_size)},
                        {bf16_range(latent, T, T == 1 ? 0 : latent_stride, 1, 0, kLatent),
                         bf16_range(rotary, T, T == 1 ? 0 : rotary_stride, 1, 0, kRotary),
                         ints_range(page_table, (uint64_t)B * max_pages), ints_range(lens, B),
                         ints_range(cu_q, B + 1LL)}),
                 FERRET_ERR_SHAPE);
  const Pages pg{page_table, max_pages, pages, page_size};
  const dim3 grid((unsigned)(((long long)T + 3) / 4));
  const auto* lat = static_cast<const uint16_t*>(latent);
  const auto* rot = static_cast<const uint16_t*>(rotary);
  if (scales != nullptr)
    hipLaunchKernelGGL((cache_write_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream, lat, latent_stride, rot,
                       rotary_stride, lens, cu_q, B, T, pg, static_cast<uint8_t*>(data),
                       static_cast<uint32_t*>(scales));
  else
    hipLaunchKernelGGL((cache_write_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream, lat, latent_stride, rot,
                       rotary_stride, lens, cu_q, B, T, pg, static_cast<uint8_t*>(data), nullptr);
  return (int)hipGetLastError();
}

extern "C" int ferret_latent_cache_read(const void* data, const void* scales, int pages, int page_size,
                                        const int32_t* page_table, const int32_t* cu_k, int B, int max_pages, int rows,
                                        void* latent, void* rotary, void* stream) {
  FERRET_REQUIRE(data && cu_k && latent && rotary, FERRET_ERR_NULL);
  const int rc = ferret_check_pages(page_table, B, max_pages, pages, page_size);
  if (rc != FERRET_OK) return rc;
  FERRET_REQUIRE(rows >= 1, FERRET_ERR_SHAPE);
  FERRET_REQUIRE(((bits(latent) | bits(rotary) | bits(data)) & 15) == 0 && (bits(scales) & 3) == 0, FERRET_ERR_ALIGN);
  FERRET_REQUIRE(!clash({Range{latent, (uint64_t)rows * kLatent * 2}, Range{rotary, (uint64_t)rows * kRotary * 2}},
                        {data_range(data, scales, pages, page_size), scale_range(scales, pages, page_size),
                         ints_range(page_table, (uint64_t)B * max_pages), ints_range(cu_k, B + 1LL)}),
                 FERRET_ERR_SHAPE);
  const Pages pg{page_table, max_pages, pages, page_size};
  const dim3 grid((unsigned)(((long long)rows + 3) / 4));
  if (scales != nullptr)
    hipLaunchKernelGGL((cache_read_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream,
                       static_cast<const uint8_t*>(data), static_cast<const uint32_t*>(scales), cu_k, B, rows, pg,
                       static_cast<uint16_t*>(latent), static_cast<uint16_t*>(rotary));
  else
    hipLaunchKernelGGL((cache_read_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream,
                       static_cast<const uint8_t*>(data), nullptr, cu_k, B, rows, pg, static_cast<uint16_t*>(latent),
                       static_cast<uint16_t*>(rotary));
  return (int)hipGetLastError();
}
