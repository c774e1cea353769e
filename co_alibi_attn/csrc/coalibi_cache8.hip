// Key / value caches held in 8 bits, on gfx950: quantising rows as they are written, and reading them back.
//
// A value is code * scale, with a scale for each kv head's blocks of 16 rows.  A block that is begun gets the least power of two
// 2^k, k >= -40, at which none of its new rows passes the format's largest code; a block that has rows keeps its scale, or
// doubles it as often as the new ones need, and its codes are halved as often.  Scaling by powers of two rounds nothing but the
// codes, so that however often a block's scale grows its int8 codes stay within one step of their values (half a step for the
// last rounding, and less than another half for all earlier ones together, whose steps were a half, a quarter, ... of it) and its
// e4m3 codes within the format's own half step, below its smallest normal number within one of its smallest steps.
//   A new value that is not finite, or too large for the largest scale, makes its block's scale NaN, and with it all that is
// read from the block, until its first row is written again.
//
// Both are copies, a wavefront per block, kv head and cache: its table entry, page and scale are looked up once, the largest new
// value is found and applied without leaving the wavefront, and no two wavefronts write one scale.  Measured in a replayed graph:
//   append, 8 prompts of 14730 rows together (8 kv heads, D 128, bf16 to int8): 17.4 us for 60.3 MB, 3.5 TB/s (a copy reaches 4.9:
//     12.4 us); the loads have to arrive before the first code is known, and a wavefront has one block's in flight;
//   append, one token for each of 16 sequences: 4.1 us, of which an empty kernel takes 2.1;
//   read, 8 sequences of up to 4096 rows (8 kv heads, D 128, e4m3 to bf16): 34.6 us for 178 MB, 5.2 TB/s; one wavefront per 64
//     pieces without blocks, with a table entry and a scale for each lane, took 54;
//   read, 500 rows of 12 heads to fp32: 3.9 us.
#include <algorithm>

#include "coalibi_codes.h"
#include "coalibi_kernels.h"
#include "coalibi_wave.h"

namespace coalibi {

namespace {

constexpr int kCacheThreads = 256;
constexpr int kCacheWaves = kCacheThreads / 64;

template <typename T>
__device__ __forceinline__ f32x8 load8(const T* p) {
  f32x8 x;
  const auto v = ld_vec8(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
  return x;
}

// The least k with x <= 2^k times the format's largest code, for finite x >= 0 given as its bits (subnormals as the smallest
// exponent).
template <typename F>
__device__ __forceinline__ int least_exponent(unsigned bits) {
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
  constexpr int e = __is_same(F, E4M3) ? 8 : 6;
  constexpr unsigned m = __is_same(F, E4M3) ? 0x600000u : 0x7e0000u;
  return (int)(bits >> 23) - 127 - e + ((bits & 0x7fffffu) > m ? 1 : 0);
}
constexpr int kLeastExponent = -40, kMostExponent = 40;

// One wavefront per block of 16 rows that gets new ones, kv head and cache: 8 elements a lane and piece, a piece's row the
// block's row.
template <typename T, typename F, int D>
__global__ __launch_bounds__(kCacheThreads) void coalibi_append8_kernel(Append8Args a8) {
  const AppendArgs& a = a8.t;
  constexpr int PPR = D / 8;                                 // pieces per row
  constexpr int N = kScaleRows * PPR < 64 ? 1 : kScaleRows * PPR / 64;  // pieces per lane
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long id = (long long)blockIdx.x * kCacheWaves + wave;
  const int h = (int)(id % a.Hkv);
  const long long block_no = id / a.Hkv;
  const bool value = blockIdx.z != 0;
  const Layout& from = value ? a.vl : a.kl;
  const Layout& to = value ? a.vcl : a.kcl;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const long long len = a.seq_lens[b];
    const int n = a.counts == nullptr ? a.N : min(max(a.counts[b], 0), a.N);
    // The new rows are cache rows [lo, hi); the block has `had` rows before them.
    const int lo = (int)min(max(len, 0ll), (long long)a.capacity);
    const int hi = (int)max(min(len + n, (long long)a.capacity), 0ll);
    const long long at = (long long)(lo / kScaleRows + block_no) * kScaleRows;
    if (at >= hi) continue;
    const int row0 = (int)at, had = max(lo - row0, 0), end = min(hi - row0, kScaleRows);
    int unit = b, in_unit = row0;
    if (a.place.table != nullptr) {
      unit = a.place.table[(size_t)b * a.place.table_stride + (row0 >> a.place.page_shift)];
      if (unit < 0 || unit >= a.place.units) continue;
      in_unit = row0 & ((1 << a.place.page_shift) - 1);
    }
    const T* const src = static_cast<const T*>(value ? a.v : a.k) + (size_t)b * from.b + (size_t)h * from.h;
    char* const dst = static_cast<char*>(value ? a.vc : a.kc) + (size_t)unit * to.b + (size_t)h * to.h + (size_t)in_unit * D;
    float* const scale = (value ? a8.vs + (size_t)unit * a8.vsb + (size_t)h * a8.vsh : a8.ks + (size_t)unit * a8.ksb + (size_t)h * a8.ksh) +
                         in_unit / kScaleRows;

    // The pieces: new ones (their values), old ones (their codes), others.
    f32x8 x[N];
    u32x2 old[N];
    bool fresh[N], held[N];
    unsigned top = 0;
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = lane + 64 * i, r = p / PPR, col = p % PPR * 8;
      held[i] = r < had;
      fresh[i] = r >= had && r < end;
      x[i] = f32x8{};
      old[i] = u32x2{};
      if (held[i]) {
        old[i] = *reinterpret_cast<const u32x2*>(dst + r * D + col);
      } else if (fresh[i]) {
        const int ni = (int)(row0 + r - len);
        const int s = a.rows == nullptr ? ni : a.rows[(size_t)b * a.N + ni];
        fresh[i] = s >= 0 && s < a.T;
        if (fresh[i]) x[i] = load8(src + (size_t)s * from.r + col);
      }
      any |= fresh[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = fabsf(x[i][e]);
        top = max(top, __builtin_bit_cast(unsigned, y));
      }
    }
    if (!__any(any)) continue;
    const float was = had > 0 ? *scale : 0.f;
    top = wave_max(top);

    int grow = 0;  // doublings of the scale that the block had
    float now;
    if (had > 0) {
      const unsigned t = __builtin_bit_cast(unsigned, was * F::kMost);
      grow = max((int)(top >> 23) - (int)(t >> 23) + ((top & 0x7fffffu) > (t & 0x7fffffu) ? 1 : 0), 0);
      now = was >= kScaleLeast && was <= kScaleMost ? ldexpf(was, grow) : __builtin_nanf("");
    } else {
      const int k = max(least_exponent<F>(top), kLeastExponent);
      now = k > kMostExponent ? __builtin_nanf("") : ldexpf(1.f, k);
    }
    const bool fine = now <= kScaleMost && top < 0x7f800000u;
    if (!fine) now = __builtin_nanf("");
    // (A block whose scale is no power of two came from elsewhere.)
    const bool two = (__builtin_bit_cast(unsigned, now) & 0x7fffffu) == 0;
    const float inv = 1.f / now, shrink = ldexpf(1.f, -grow);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = lane + 64 * i, r = p / PPR, col = p % PPR * 8;
      f32x8 y{};
      if (fresh[i]) {
        if (fine) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = two ? x[i][e] * inv : x[i][e] / now;
        }
      } else if (held[i] && fine && grow > 0) {
        y = from_codes<F>(old[i]) * shrink;
      } else {
        continue;
      }
      *reinterpret_cast<u32x2*>(dst + r * D + col) = to_codes<F>(y);
    }
    if (lane == 0) *scale = now;
  }
}

// Rows [first, first + n) of every sequence: a wavefront per block of 16 rows, kv head and cache, whose page and scale are then its
// own, and 16 codes a lane and piece.
template <typename T, typename F, int D>
__global__ __launch_bounds__(kCacheThreads) void coalibi_read8_kernel(Read8Args a) {
  constexpr int PPR = D / 16, N = PPR * kScaleRows < 64 ? 1 : PPR * kScaleRows / 64;  // pieces per row, and per lane
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long id = (long long)blockIdx.x * kCacheWaves + wave;
  const int block = __builtin_amdgcn_readfirstlane((int)(id / a.Hkv)), h = (int)(id - (long long)block * a.Hkv);
  const bool value = blockIdx.z != 0;
  const Layout& l = value ? a.vcl : a.kcl;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const long long first = a.first == nullptr ? 0 : a.first[b];
    const long long at = (first & ~(long long)(kScaleRows - 1)) + (long long)block * kScaleRows;  // (rounded down, below 0 too)
    if (at >= first + a.N) continue;
    const int filled = min(a.seq_lens[b], a.capacity);
    T* const out = static_cast<T*>(value ? a.v : a.k) + ((size_t)b * a.Hkv + h) * a.N * D;
    float s = 0.f;
    const char* p = nullptr;
    if (at >= 0 && at < filled) {
      int unit = b, in_unit = (int)at;
      bool there = true;
      if (a.place.table != nullptr) {
        unit = a.place.table[(size_t)b * a.place.table_stride + (in_unit >> a.place.page_shift)];
        there = unit >= 0 && unit < a.place.units;
        in_unit &= (1 << a.place.page_shift) - 1;
      }
      if (there) {
        const float x = value ? a.vs[(size_t)unit * a.vsb + (size_t)h * a.vsh + in_unit / kScaleRows]
                              : a.ks[(size_t)unit * a.ksb + (size_t)h * a.ksh + in_unit / kScaleRows];
        s = x >= kScaleLeast && x <= kScaleMost ? x : __builtin_nanf("");
        p = static_cast<const char*>(value ? a.vc : a.kc) + (size_t)unit * l.b + (size_t)h * l.h + (size_t)in_unit * D;
      } else {
        s = __builtin_nanf("");
      }
    }
    const int left = p == nullptr ? 0 : (int)min(filled - at, (long long)kScaleRows);  // rows that are read
    u32x4 c[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int piece = lane + 64 * i, r = piece / PPR;
      c[i] = u32x4{};
      if (r < left) c[i] = ld16(p + piece * 16);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int piece = lane + 64 * i, r = piece / PPR;
      const long long row = at + r - first;
      if (r >= kScaleRows || row < 0 || row >= a.N) continue;
      const float f = at + r < filled ? s : 0.f;
      f32x8 x[2] = {from_codes<F>(u32x2{c[i][0], c[i][1]}), from_codes<F>(u32x2{c[i][2], c[i][3]})};
#pragma unroll
      for (int j = 0; j < 2; ++j) store8(out + row * D + piece % PPR * 16 + 8 * j, x[j] * f);
    }
  }
}

template <typename T, typename F>
hipError_t append_d(const Append8Args& a, int D, dim3 grid, hipStream_t st) {
  switch (D) {
    case 16: hipLaunchKernelGGL((coalibi_append8_kernel<T, F, 16>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 32: hipLaunchKernelGGL((coalibi_append8_kernel<T, F, 32>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 64: hipLaunchKernelGGL((coalibi_append8_kernel<T, F, 64>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 128: hipLaunchKernelGGL((coalibi_append8_kernel<T, F, 128>), grid, dim3(kCacheThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((coalibi_append8_kernel<T, F, 256>), grid, dim3(kCacheThreads), 0, st, a); break;
  }
  return hipGetLastError();
}

template <typename T, typename F>
hipError_t read_d(const Read8Args& a, dim3 grid, hipStream_t st) {
  switch (a.D) {
    case 16: hipLaunchKernelGGL((coalibi_read8_kernel<T, F, 16>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 32: hipLaunchKernelGGL((coalibi_read8_kernel<T, F, 32>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 64: hipLaunchKernelGGL((coalibi_read8_kernel<T, F, 64>), grid, dim3(kCacheThreads), 0, st, a); break;
    case 128: hipLaunchKernelGGL((coalibi_read8_kernel<T, F, 128>), grid, dim3(kCacheThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((coalibi_read8_kernel<T, F, 256>), grid, dim3(kCacheThreads), 0, st, a); break;
  }
  return hipGetLastError();
}

}  // namespace

template <typename T>
hipError_t launch_append8(const Append8Args& a, bool e4m3, int D, hipStream_t stream) {
  // N rows from anywhere in a block touch at most (N + 14) / 16 + 1 blocks.
  const long long waves = ((a.t.N + kScaleRows - 2ll) / kScaleRows + 1) * a.t.Hkv;
  const dim3 grid(static_cast<unsigned>((waves + kCacheWaves - 1) / kCacheWaves), static_cast<unsigned>(std::min(a.t.B, 65535)), 2);
  return e4m3 ? append_d<T, E4M3>(a, D, grid, stream) : append_d<T, I8>(a, D, grid, stream);
}

template <typename T>
hipError_t launch_read8(const Read8Args& a, bool e4m3, hipStream_t stream) {
  const long long waves = ((a.N + kScaleRows - 2ll) / kScaleRows + 1) * a.Hkv;
  const dim3 grid(static_cast<unsigned>((waves + kCacheWaves - 1) / kCacheWaves), static_cast<unsigned>(std::min(a.B, 65535)), 2);
  return e4m3 ? read_d<T, E4M3>(a, grid, stream) : read_d<T, I8>(a, grid, stream);
}

#define COALIBI_INST_CACHE8(T)                                                          \
  template hipError_t launch_append8<T>(const Append8Args&, bool, int, hipStream_t);    \
  template hipError_t launch_read8<T>(const Read8Args&, bool, hipStream_t);
COALIBI_INST_CACHE8(_Float16)
COALIBI_INST_CACHE8(__bf16)
COALIBI_INST_CACHE8(float)

}  // namespace coalibi
