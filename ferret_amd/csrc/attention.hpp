// What the attention kernels share: transposing LDS reads, asynchronous copies into
// LDS with the waits left to the kernel, and the softmax's constants.
#pragma once

#include "common.hpp"

namespace ferret {

// The running maximum moves only when a score passes it by more than 2^kLazy (log2
// units): the softmax terms stay <= 256 and the output is rescaled for few steps only.
constexpr float kLazy = 8.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
#define FERRET_LDS __attribute__((address_space(3)))

// Transposing LDS reads.  Each group of 16 lanes reads a block: lane 4j + i (of 16)
// points at elements 4i .. 4i+3 of row j (16-bit, 4 rows), lane 2j + i at bytes 8i ..
// 8i+7 of row j (8-bit, 8 rows); lane c receives column c, rows in order.
__device__ __forceinline__ u32x2 lds_tr16(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((FERRET_LDS s16x4*)p));
}
__device__ __forceinline__ u32x2 lds_tr8(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((FERRET_LDS i32x2*)p));
}

// Global -> LDS copies of 16 and 4 bytes per lane: lane l fills `lds_at` + size * l
// (an LDS address, the same in all lanes) from base + off.  Written as assembly
// because the compiler, which tracks the builtin's loads, waits for all of them
// before every transposing LDS read; the waits here are the kernel's own
// (wait_vmcnt).  No register is loaded, so nothing of theirs can be reused early; M0,
// a register that the compiler reserves, has no other user in these kernels.
__device__ __forceinline__ void dma_16(const uint8_t* base, int off, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_at)
               : "memory");
}
__device__ __forceinline__ void dma_4(const uint32_t* base, int off, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds_at)
               : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) { return (uint32_t)(uintptr_t)(FERRET_LDS uint8_t*)p; }

// All LDS accesses of the work-group so far are done; loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Maximum over lanes l, l ^ 16, l ^ 32, l ^ 48, in all of them.
__device__ __forceinline__ float rows_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

}  // namespace ferret
