// Reductions over a wavefront by DPP moves and lane swaps (a shuffle takes an LDS round trip a step).
#pragma once
#include "coalibi_common.h"

namespace coalibi {

namespace {

typedef unsigned long long u64;

// The number of a lane's partner in step S of six that join 1, 2, 4, ..., 32 lanes, of which those of a group hold the same.
template <int S>
__device__ __forceinline__ unsigned partner(unsigned x) {
  if constexpr (S < 4) {  // quad_perm [1, 0, 3, 2] and [2, 3, 0, 1], row_half_mirror, row_mirror
    constexpr int ctrl = S == 0 ? 0xb1 : S == 1 ? 0x4e : S == 2 ? 0x141 : 0x140;
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, false);
  } else if constexpr (S == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int S>
__device__ __forceinline__ u64 partner(u64 x) {
  return (u64)partner<S>((unsigned)(x >> 32)) << 32 | partner<S>((unsigned)x);
}
template <int S>
__device__ __forceinline__ float partner(float x) {
  return __builtin_bit_cast(float, partner<S>(__builtin_bit_cast(unsigned, x)));
}
template <int S>
__device__ __forceinline__ double partner(double x) {
  return __builtin_bit_cast(double, partner<S>(__builtin_bit_cast(u64, x)));
}
template <int S = 0, typename X>
__device__ __forceinline__ X wave_max(X x) {
  if constexpr (S == 6) {
    return x;
  } else {
    const X y = partner<S>(x);
    return wave_max<S + 1>(y > x ? y : x);
  }
}
template <int S = 0>
__device__ __forceinline__ double wave_sum(double x) {
  if constexpr (S == 6)
    return x;
  else
    return wave_sum<S + 1>(x + partner<S>(x));
}

}  // namespace

}  // namespace coalibi
