// Sampling the next token from a row of logits on gfx950: temperature, top-k, top-p and min-p from a given
// uniform number.
//
// With the tokens in order (logit descending, then index ascending) and weights w_i = exp((x_i - max x) / T):
//   top-k keeps the first k;  top-p of those the ones whose weights before them sum to less than p times
//   the sum of the top-k's;  min-p of those the ones with w_i >= min_p (max w is 1).  What is kept is a prefix
//   and never empty.  The token is the first whose inclusive sum of weights exceeds u times the kept sum.
//
// Nothing is sorted.  Every step is a search for a position along that order, by count or by weight, and a
// position is found digit by digit of the logit's order-preserving integer key (radix select): a histogram
// of one digit, a scan from its largest value, and the next digit within the bin that holds the
// position.  Tokens of one key have one weight, so the position among them is a division.
//   Weights are integers, 2^mass_bits * w rounded (mass_bits = 62 - ceil(log2 V), 46 for 50304 tokens): integer
// sums do not depend on the order in which atomics add, and the same call gives the same token.  The rounding
// moves a border by less than V * 2^-63 of the largest weight.  They are computed in fp64: with fp32
// exponentials (2^-22) a border between 50304 tokens would move past the uniform number in one draw of about a
// thousand.
#include <cmath>

#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

typedef unsigned long long u64;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;

// A logit's key: unsigned integers in the logits' order, with -0 taken for +0.
template <typename T>
struct Key {
  static constexpr int kBits = 8 * sizeof(T);
  static constexpr unsigned kSign = 1u << (kBits - 1), kMask = kSign | (kSign - 1);
  static __device__ __forceinline__ unsigned of(T x) {
    unsigned u;
    if constexpr (sizeof(T) == 4)
      u = __builtin_bit_cast(unsigned, x);
    else
      u = __builtin_bit_cast(unsigned short, x);
    if (u == kSign) u = 0;
    return u & kSign ? ~u & kMask : u | kSign;
  }
  static __device__ __forceinline__ float value(unsigned k) {
    const unsigned u = k & kSign ? k & ~kSign : ~k & kMask;
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(float, u);
    else
      return static_cast<float>(__builtin_bit_cast(T, static_cast<unsigned short>(u)));
  }
};

struct SampleLds {
  unsigned cnt[kBins];
  u64 mass[kBins];
  unsigned wcnt[kSampleWaves];
  u64 wmass[kSampleWaves];
  int bin;
  u64 before_cnt, before_mass;
  u64 sum;
  unsigned key;
  int flag, token;
};

// The weights of one row.
struct Weights {
  double top, temp, one;
  __device__ __forceinline__ double w(float x) const {
    const double d = static_cast<double>(x) - top;
    return x == static_cast<float>(top) ? 1.0 : d == -__builtin_inf() ? 0.0 : exp(d / temp);
  }
  __device__ __forceinline__ u64 mass(double w) const { return static_cast<u64>(w * one + 0.5); }
};

// The histogram of the digit at bits [shift, shift + kDigitBits) of the keys, over the tokens whose key bits
// from `top` on are `prefix`'s; ends with a barrier.  Returns this thread's part of the mass of the tokens
// with w >= min_p.
template <typename T>
__device__ u64 histogram(SampleLds& s, const T* row, int V, unsigned prefix, int top, int shift, const Weights& ws,
                         double min_p) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kBins; i += kSampleThreads) s.cnt[i] = 0, s.mass[i] = 0;
  __syncthreads();
  u64 heavy = 0;
  for (int i = tid; i < V; i += kSampleThreads) {
    const T x = row[i];
    const unsigned k = Key<T>::of(x);
    if (top < Key<T>::kBits && (k ^ prefix) >> top != 0) continue;
    const double w = ws.w(static_cast<float>(x));
    const u64 m = ws.mass(w);
    const int bin = k >> shift & (kBins - 1);
    atomicAdd(&s.cnt[bin], 1u);
    if (m != 0) atomicAdd(&s.mass[bin], m);
    if (w >= min_p) heavy += m;
  }
  __syncthreads();
  return heavy;
}

// The bin that holds position `pos` (counted by tokens, or by mass with by_mass) among the histogram's bins
// from the largest down, and what lies before it, into s.bin / s.before_*: each thread scans two bins.
__device__ void find_bin(SampleLds& s, u64 pos, bool by_mass) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b0 = kBins - 1 - 2 * tid, b1 = b0 - 1;
  const u64 c0 = s.cnt[b0], c1 = s.cnt[b1], m0 = s.mass[b0], m1 = s.mass[b1];
  u64 c = c0 + c1, m = m0 + m1;
  for (int off = 1; off < 64; off <<= 1) {
    const u64 oc = __shfl_up(c, off, 64), om = __shfl_up(m, off, 64);
    if (lane >= off) c += oc, m += om;
  }
  if (lane == 63) s.wcnt[wave] = (unsigned)c, s.wmass[wave] = m;
  __syncthreads();
  for (int w = 0; w < wave; ++w) c += s.wcnt[w], m += s.wmass[w];
  // [before, before + own) of each of the two bins.
  u64 cb = c - c0 - c1, mb = m - m0 - m1;
  for (int e = 0; e < 2; ++e) {
    const u64 oc = e == 0 ? c0 : c1, om = e == 0 ? m0 : m1;
    const u64 before = by_mass ? mb : cb, own = by_mass ? om : oc;
    if (pos >= before && pos - before < own) {
      s.bin = e == 0 ? b0 : b1;
      s.before_cnt = cb;
      s.before_mass = mb;
    }
    cb += oc;
    mb += om;
  }
  __syncthreads();
}

struct Place {
  unsigned key;
  u64 before_cnt, before_mass;  // of the tokens with larger keys
};

template <typename T>
__device__ Place locate(SampleLds& s, const T* row, int V, u64 pos, bool by_mass, const Weights& ws) {
  Place p{0, 0, 0};
  for (int top = Key<T>::kBits; top > 0; top -= kDigitBits) {
    const int shift = max(top - kDigitBits, 0);
    // The last digit reaches above `top` where the key's bits are no multiple of a digit's; the tokens agree there.
    histogram(s, row, V, p.key, top, shift, ws, 0.0);
    find_bin(s, pos, by_mass);
    const unsigned digit = s.bin;
    p.key = (p.key & ~((unsigned)(kBins - 1) << shift)) | digit << shift;
    p.before_cnt += s.before_cnt;
    p.before_mass += s.before_mass;
    pos -= by_mass ? s.before_mass : s.before_cnt;
    __syncthreads();
  }
  return p;
}

__device__ u64 block_sum(u64 x, SampleLds& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  if (lane == 0) s.wmass[wave] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < kSampleWaves; ++w) x += s.wmass[w];
  __syncthreads();
  return x;
}

// The index of the token of key `key` that `nth` others of that key precede.
template <typename T>
__device__ int nth_token(SampleLds& s, const T* row, int V, unsigned key, u64 nth) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (V + kSampleThreads - 1) / kSampleThreads * 64, lo = min(wave * per, V), hi = min(lo + per, V);
  unsigned n = 0;
  for (int i = lo + lane; i < hi; i += 64) n += Key<T>::of(row[i]) == key;
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  if (lane == 0) s.wcnt[wave] = n;
  __syncthreads();
  u64 before = 0;
  for (int w = 0; w < wave; ++w) before += s.wcnt[w];
  if (nth >= before && nth < before + n) {
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const int i = i0 + lane;
      const bool is = i < hi && Key<T>::of(row[i]) == key;
      const u64 mask = __ballot(is);
      if (is && before + __popcll(mask & ((1ull << lane) - 1)) == nth) s.token = i;
      before += __popcll(mask);
    }
  }
  __syncthreads();
  return s.token;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void coalibi_sample_kernel(SampleArgs a) {
  __shared__ SampleLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const T* const row = static_cast<const T*>(a.logits) + b * a.row_stride;
  const double temp = a.temperature != nullptr ? static_cast<double>(a.temperature[b]) : a.temperature_all;
  const int top_k = a.top_k != nullptr ? a.top_k[b] : a.top_k_all;
  const double top_p = a.top_p != nullptr ? static_cast<double>(a.top_p[b]) : a.top_p_all;
  const double min_p = a.min_p != nullptr ? static_cast<double>(a.min_p[b]) : a.min_p_all;
  const double uni = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[b]
                                    : static_cast<double>(static_cast<const float*>(a.uniforms)[b]);
  // The largest key, and whether a logit is NaN.
  unsigned kmax = 0;
  bool nan = false;
  for (int i = tid; i < a.V; i += kSampleThreads) {
    const T x = row[i];
    nan |= static_cast<float>(x) != static_cast<float>(x);
    kmax = max(kmax, Key<T>::of(x));
  }
  for (int off = 32; off > 0; off >>= 1) kmax = max(kmax, (unsigned)__shfl_xor((int)kmax, off, 64));
  if (lane == 0) s.wcnt[wave] = kmax;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < kSampleWaves; ++w) kmax = max(kmax, s.wcnt[w]);
  const float top = Key<T>::value(kmax);
  __syncthreads();
  if (nan || top == kNegInf) {
    if (tid == 0) a.tokens[b] = -1;
    return;
  }
  unsigned key = kmax;
  u64 nth = 0;
  if (temp > 0.0) {  // else (0, negative, NaN): the first of the largest logits
    const Weights ws{static_cast<double>(top), temp, static_cast<double>(1ull << a.mass_bits)};
    const u64 heavy = block_sum(histogram(s, row, a.V, 0u, Key<T>::kBits, Key<T>::kBits - kDigitBits, ws, min_p), s);
    u64 all = 0;
    for (int i = tid; i < kBins; i += kSampleThreads) all += s.mass[i];
    all = block_sum(all, s);
    u64 kept = all;
    if (top_k > 0 && top_k < a.V) {
      const Place p = locate(s, row, a.V, top_k - 1, false, ws);
      kept = p.before_mass + (top_k - p.before_cnt) * ws.mass(ws.w(Key<T>::value(p.key)));
    }
    u64 cut = kept;
    if (top_p < 1.0) {
      // Tokens are kept while the mass before them is below the bound: up to the one at its last unit.
      const double bound = fmax(ceil(top_p * static_cast<double>(kept)), 1.0);
      const u64 pos = static_cast<u64>(bound) - 1;
      if (pos < all) {
        const Place p = locate(s, row, a.V, pos, true, ws);
        const u64 w = ws.mass(ws.w(Key<T>::value(p.key)));
        cut = min(cut, p.before_mass + ((pos - p.before_mass) / w + 1) * w);
      }
    }
    if (min_p > 0.0) cut = min(cut, max(heavy, ws.mass(1.0)));
    const double at = uni > 0.0 ? uni * static_cast<double>(cut) : 0.0;
    const u64 pos = at < static_cast<double>(cut) ? min(static_cast<u64>(at), cut - 1) : cut - 1;
    const Place p = locate(s, row, a.V, pos, true, ws);
    key = p.key;
    nth = (pos - p.before_mass) / ws.mass(ws.w(Key<T>::value(key)));
  }
  const int token = nth_token(s, row, a.V, key, nth);
  if (tid == 0) a.tokens[b] = token;
}

}  // namespace

template <typename T>
hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((coalibi_sample_kernel<T>), dim3(a.B), dim3(kSampleThreads), 0, stream, a);
  return hipGetLastError();
}

template hipError_t launch_sample<_Float16>(const SampleArgs&, hipStream_t);
template hipError_t launch_sample<__bf16>(const SampleArgs&, hipStream_t);
template hipError_t launch_sample<float>(const SampleArgs&, hipStream_t);

}  // namespace coalibi
