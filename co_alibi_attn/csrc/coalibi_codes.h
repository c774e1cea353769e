// Codes of 8 bits (e4m3, or int8 in [-127, 127]) from and to fp32, eight at a time.
#pragma once
#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

template <typename F>
__device__ __forceinline__ f32x8 from_codes(u32x2 c) {
  f32x8 x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (__is_same(F, E4M3)) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
      x[4 * i] = lo[0];
      x[4 * i + 1] = lo[1];
      x[4 * i + 2] = hi[0];
      x[4 * i + 3] = hi[1];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = static_cast<float>(static_cast<signed char>(c[i] >> 8 * e));
    }
  }
  return x;
}

// The nearest codes, ties to even, of values that no more than a rounding puts past the largest code: such ones become it.
template <typename F>
__device__ __forceinline__ u32x2 to_codes(f32x8 x) {
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (__is_same(F, E4M3)) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
      c[i] = (unsigned)w;
    } else {
      // In the last byte of 1.5 * 2^23 + x.
      unsigned w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = __builtin_amdgcn_fmed3f(x[4 * i + e], -F::kMost, F::kMost) + 0x1.8p23f;
        w[e] = __builtin_bit_cast(unsigned, y);
      }
      const unsigned lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(w[3], w[2], 0x04000c0cu);
      c[i] = lo | hi;
    }
  }
  return c;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, f32x8 x) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<typename Mfma<T>::vec8*>(p) = Mfma<T>::pack(x);
  }
}

}  // namespace

}  // namespace coalibi
