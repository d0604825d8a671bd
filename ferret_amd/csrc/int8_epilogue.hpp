// What the int8 products do with a whole sum.
#pragma once

#include "common.hpp"
#include "int8_plan.hpp"

namespace ferret {
namespace i8 {

// Four outputs of token m (scale sa) from channel n on, each step rounded by itself: a
// contracted one would change bits with the variant that the compiler contracts.
__device__ __forceinline__ u32x2 four_outputs(const Args& p, int m, int n, float sa, i32x4 sum) {
#pragma clang fp contract(off)
  const f32x4 sb = *reinterpret_cast<const f32x4*>(p.sb + n);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)sum[i] * sa * sb[i];
  if (p.residual != nullptr) {
    const u32x2 r = *reinterpret_cast<const u32x2*>(p.residual + (size_t)m * p.N + n);
    v[0] += __uint_as_float(r[0] << 16);
    v[1] += __uint_as_float(r[0] & 0xffff0000u);
    v[2] += __uint_as_float(r[1] << 16);
    v[3] += __uint_as_float(r[1] & 0xffff0000u);
  }
  return u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

}  // namespace i8
}  // namespace ferret
