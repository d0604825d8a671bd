// The paged latent cache: its row formats, and where a token's row stands.
//
// A row is the 512 normed key-value latents of one token and its 64 rotary key
// values.  bf16: 576 values, 1152 bytes.  e4m3: 512 codes, then the rotary
// values as bf16, 640 bytes; and one exponent byte per 128 latents in an array of
// its own (4 bytes a row).  A byte b stands for 2^(b - 127), b >= kMinByte, so
// that every code times its scale is a normal bf16 value: reading back is exact.
// Powers of two cost nothing in precision (codes are floating-point numbers too)
// and let v_cvt_scalef32_pk_bf16_fp8 widen and scale in one instruction.
//
// Pages hold page_size rows (a multiple of 16); page_table [B, max_pages] names
// the pages of a sequence in order.  An entry outside [0, pages) stands for no
// page: writes to it are dropped, reads give zeros, attention leaves its keys out.
#pragma once

#include "common.hpp"
#include "latent_plan.hpp"
#include "ranges.hpp"

namespace ferret {

constexpr int kLatent = 512, kRotary = 64;
constexpr int kRowBf16 = 2 * (kLatent + kRotary);  // bytes
constexpr int kRowE4m3 = kLatent + 2 * kRotary;
constexpr int kMinByte = 16;

struct Pages {
  const int32_t* table;  // [B, max_pages]
  int max_pages, pages, page_size;
};

// What the cache's two arrays and the page table span.
inline Range data_range(const void* data, const void* scales, int pages, int page_size) {
  return {data, (uint64_t)pages * page_size * (scales != nullptr ? kRowE4m3 : kRowBf16)};
}
inline Range scale_range(const void* scales, int pages, int page_size) {
  return {scales, (uint64_t)pages * page_size * 4};
}
inline Range ints_range(const int32_t* at, uint64_t n) { return {at, 4 * n}; }

// The row number of position `pos` of sequence b in the cache, -1 for no row.
__device__ __forceinline__ long long cache_row(const Pages& p, int b, int pos) {
  if (pos < 0) return -1;
  const int page = pos / p.page_size;
  if (page >= p.max_pages) return -1;
  return page_row(p.table[(long long)b * p.max_pages + page], p.pages, p.page_size, pos - page * p.page_size);
}

// The sequence that packed row t belongs to: the number of sequences that end at
// or before it, counted by the lanes of a wave together (one load deep for up to
// 64 sequences, where a search by halves would be six loads deep).  `starts`
// [B + 1] ascends; B where t stands behind the last sequence.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ starts, int B, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b = 0; b < B; b += 64) {
    const bool before = b + lane < B && starts[b + lane + 1] <= t;
    n += __popcll(__ballot(before));
  }
  return n;
}

}  // namespace ferret
