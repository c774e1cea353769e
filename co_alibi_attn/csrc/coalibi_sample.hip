// Sampling the next token from a row of logits on gfx950: temperature, top-k, top-p and min-p from a given
// uniform number.
//
// With the tokens in order (logit descending, then index ascending) and weights w_i = exp((x_i - max x) / T):
//   top-k keeps the first k;  top-p of those the ones whose weights before them sum to less than p times
//   the sum of the top-k's;  min-p of those the ones with w_i >= min_p (max w is 1).  What is kept is a prefix
//   and never empty.  The token is the first whose inclusive sum of weights exceeds u times the kept sum.
// So every step asks for a position along that order, by count or by weight, and nothing needs the whole order.
//
// Weights are integers, 2^mass_bits * w rounded (mass_bits = min(50, 62 - ceil(log2 V)), 46 for 50304 tokens):
// integer sums do not depend on the order in which atomics add, and the same call gives the same token.  The
// rounding moves a border by less than V * 2^-(mass_bits + 1) of the largest weight.  They are computed in fp64: with
// fp32 exponentials a border between 50304 tokens would move past the uniform number in one draw of about a
// thousand.
//
// One work-group per row, passes over it from L2 after the first.  What bounds it, captured: 1 row of 50304 fp32 with top-k
// 15.2 us, the latency of two passes and of the steps between; 64 rows (bf16) 16.8 us where top-k leaves a list.  By the
// histogram a row's fp64 weights and LDS atomics on one CU, whatever the batch: 1 row 36 us, 64 rows 40, 64 rows of 131072 fp32
// 79, 256 of them 102 (134 MB, 26 us at a copy's rate); with min-p, whose list saves the histogram, 256 rows of 131071 69.
//   1. the largest logit;
//   2. short lists: where top-k (or min-p) leaves few tokens, those above a bound are gathered in LDS -- for top-k the
//      k-th largest of the threads' own maxima, below which no token of the first k lies -- and all positions are
//      found among them;
//   3. otherwise a histogram of the weights over 2048 bins of the logits' distance from the largest.  Its sums bound every
//      position to a bin or two; the tokens of those bins are gathered and the positions found among them;
//   4. where a list does not fit (many equal logits), radix select: positions are found digit by digit of the logit's
//      order-preserving integer key, with a histogram per digit, and among equal tokens by division.
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
static_assert(kBins == 2 * kSampleThreads, "a thread scans two bins");
constexpr int kMaxList = 2048;
constexpr int kPerThread = kMaxList / kSampleThreads;  // listed tokens
// Largest top-k that is tried as a list.  Among 1024 threads' maxima the bound for k leaves about -1024 ln(1 - k / 1024)
// tokens in random order: 1.2 k at 350, 1.6 k at 700.  64 rows of 50304, us: k 600 17.8, 780 19.5 by the list; by the
// histogram 36.7, and 43.8 where a list of 900 is tried first and does not fit.
constexpr int kMaxListK = 800;
constexpr int kIndexBits = 20;
static_assert(kMaxVocab <= 1 << kIndexBits, "an index fits an entry");

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
__device__ __forceinline__ unsigned key32(float x) { return Key<float>::of(x); }

// A listed token: its bin (larger logits first), key and index, complemented so that the order of the tokens is the
// descending order of the words, and its weight.
struct Entry {
  u64 word;
  u64 mass;
};
__device__ __forceinline__ u64 entry_word(int bin, float x, int i) {
  return (u64)(0xfffu - bin) << 52 | (u64)key32(x) << kIndexBits | ((1u << kIndexBits) - 1 - i);
}
__device__ __forceinline__ float entry_logit(u64 word) { return Key<float>::value((unsigned)(word >> kIndexBits)); }
__device__ __forceinline__ int entry_index(u64 word) { return (1 << kIndexBits) - 1 - (int)(word & ((1u << kIndexBits) - 1)); }

// An entry's place: what lies before it in the row, by count and by mass.
struct Listed {
  u64 before_cnt, before_mass, mass;
  int token;  // -1: no entry
};

constexpr int kRounds = 8;  // of kth_of_threads
constexpr int kSums = 3;    // block_sum calls on one way through the kernel

struct SampleLds {
  u64 mass[kBins];  // a histogram's bins; then what lies before each
  unsigned cnt[kBins];
  unsigned cursor[kBins];
  u64 list[kMaxList];       // the words of the listed tokens, as found
  Entry grouped[kMaxList];  // by bin
  u64 prefix[kMaxList];     // the masses before each grouped entry
  double exp2_table[32];
  u64 wmass[kSampleWaves];
  unsigned wcnt[kSampleWaves];
  unsigned low;  // key of the smallest logit above -inf
  u64 round[kRounds], sum[kSums];  // zero at the start
  int bin;
  u64 before_cnt, before_mass, list_mass;
  int listed, token, found;
  Listed at;
};

// 2^(i / 32), rounded to fp64.
__device__ const double kExp2Table[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// The weights of one row: 2^(y / 32) with y = (x - max) * 32 log2(e) / T.
struct Weights {
  float top;          // the largest logit
  double top64, c;    // c = 32 log2(e) / T
  double reach;       // logits further than this below the largest have weight 0; fp64, as fp32 holds neither the
                      // distance of any two logits nor this at every temperature
  double one;         // 2^mass_bits
  const double* table;  // 2^mass_bits * 2^(i / 32)

  // 2^mass_bits * w, before its rounding to an integer: y = i + r with an integer i and |r| <= 1/2, 2^(r/32) by its
  // series up to r^5 (the next term is below 2^-48 of it).
  __device__ __forceinline__ double scaled(float x) const {
    const double d = static_cast<double>(x) - top64;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer, in the low bits
    const double t = fma(d, c, magic);
    const int i = static_cast<int>(static_cast<unsigned>(__builtin_bit_cast(u64, t)));
    const double r = fma(d, c, magic - t);
    constexpr double k = 0.69314718055994530942 / 32;
    double p = fma(r, k * k * k * k * k / 120, k * k * k * k / 24);
    p = fma(p, r, k * k * k / 6);
    p = fma(p, r, k * k / 2);
    p = fma(p, r, k);
    p = fma(p, r, 1.0);
    // The table's entry times 2^(i >> 5), through its exponent: the result is normal where it is used.
    const u64 e = __builtin_bit_cast(u64, table[i & 31]) + ((u64)(unsigned)((i >> 5) << 20) << 32);
    const double w = p * __builtin_bit_cast(double, e);
    return x == top ? one : d >= -reach ? w : 0.0;  // 0 also for -inf, and for what is below a +inf
  }
  static __device__ __forceinline__ u64 mass(double scaled) {
    return __builtin_bit_cast(u64, scaled + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: scaled <= 2^50
  }
  __device__ __forceinline__ u64 operator()(float x) const { return mass(scaled(x)); }
};

// f(x, index) over the row, each thread its own tokens, U loads of 16 bytes in flight (few copies of a long f).  The
// tokens before the row's first 16-byte boundary and after its last go one by one.
template <int U, typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, int V, const F& f) {
  constexpr int VEC = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const int head = min((int)(-reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T), V), n = (V - head) / VEC;
  const vec* const v = reinterpret_cast<const vec*>(row + head);
  for (int j = threadIdx.x; j < n; j += U * kSampleThreads) {
    vec x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = v[min(j + u * kSampleThreads, n - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u == 0 || j + u * kSampleThreads < n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(static_cast<T>(x[u][e]), head + (j + u * kSampleThreads) * VEC + e);
  }
  const int t = threadIdx.x, i = t < head ? t : n * VEC + t;
  if (i < V) f(row[i], i);
}

// act(x, index) for the tokens with pred(x), few of them: the tests of 32 tokens first, then the ones that passed (one
// copy of act, where a branch per token makes the kernel outgrow the instruction cache).
template <typename T, typename P, typename A>
__device__ __forceinline__ void for_row_if(const T* row, int V, const P& pred, const A& act) {
  constexpr int VEC = 16 / (int)sizeof(T), U = 32 / VEC;
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const int head = min((int)(-reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T), V), n = (V - head) / VEC;
  const vec* const v = reinterpret_cast<const vec*>(row + head);
  for (int j = threadIdx.x; j < n; j += U * kSampleThreads) {
    vec x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = v[min(j + u * kSampleThreads, n - 1)];
    unsigned hit = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u == 0 || j + u * kSampleThreads < n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) hit |= pred(static_cast<T>(x[u][e])) ? 1u << (u * VEC + e) : 0u;
    for (; hit != 0; hit &= hit - 1) {
      const int bit = __ffs(hit) - 1, i = head + (j + bit / VEC * kSampleThreads) * VEC + bit % VEC;
      act(row[i], i);
    }
  }
  const int t = threadIdx.x, i = t < head ? t : n * VEC + t;
  if (i < V && pred(row[i])) act(row[i], i);
}

// The sum over the work-group, each call with a slot of its own (integers: any order gives the same).
__device__ __forceinline__ u64 block_sum(u64 x, SampleLds& s, int slot) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  if ((threadIdx.x & 63) == 0) atomicAdd(&s.sum[slot], x);
  __syncthreads();
  return s.sum[slot];
}

// ------------------------------------------------------------------ positions in a list

// Each of the n entries of s.list learns what lies before it: the entries are grouped by bin, and within their bin compared
// with one another.  Before a bin lies what s.mass / s.cnt say, or with `whole` (the list is all that counts) what the list
// holds before it.  Thread t has the entries t, t + kSampleThreads, ... in `out`, and their weights' sum in s.list_mass.
__device__ __forceinline__ void place_listed(SampleLds& s, int n, bool whole, const Weights& ws, Listed (&out)[kPerThread]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto bin_of = [](u64 word) { return 0xfff - (int)(word >> 52); };
  s.cursor[2 * tid] = s.cursor[2 * tid + 1] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kSampleThreads) atomicAdd(&s.cursor[bin_of(s.list[i])], 1u);
  __syncthreads();
  const unsigned n0 = s.cursor[2 * tid], n1 = s.cursor[2 * tid + 1];
  unsigned c = n0 + n1;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned o = __shfl_up(c, off, 64);
    if (lane >= off) c += o;
  }
  if (lane == 63) s.wcnt[wave] = c;
  __syncthreads();
  unsigned w = lane < wave ? s.wcnt[lane & (kSampleWaves - 1)] : 0;
#pragma unroll
  for (int off = kSampleWaves / 2; off > 0; off >>= 1) w += __shfl_xor(w, off, kSampleWaves);
  c += __shfl(w, 0, 64) - n0 - n1;  // entries of the bins before this thread's
  s.cursor[2 * tid] = c;
  s.cursor[2 * tid + 1] = c + n0;
  __syncthreads();
  for (int i = tid; i < n; i += kSampleThreads) {
    const u64 word = s.list[i];
    // A bin's cursor ends at the next bin's start.
    s.grouped[atomicAdd(&s.cursor[bin_of(word)], 1u)] = {word, ws(entry_logit(word))};
  }
  __syncthreads();
  // The masses before each entry: kPerThread consecutive ones a thread.
  u64 own[kPerThread], m = 0;
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const int i = tid * kPerThread + u;
    own[u] = i < n ? s.grouped[i].mass : 0;
    m += own[u];
  }
  const u64 total = m;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 o = __shfl_up(m, off, 64);
    if (lane >= off) m += o;
  }
  if (lane == 63) s.wmass[wave] = m;
  __syncthreads();
  u64 wm = lane < wave ? s.wmass[lane & (kSampleWaves - 1)] : 0;
#pragma unroll
  for (int off = kSampleWaves / 2; off > 0; off >>= 1) wm += __shfl_xor(wm, off, kSampleWaves);
  m += __shfl(wm, 0, 64);
  if (tid == kSampleThreads - 1) s.list_mass = m;
  m -= total;
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    if (tid * kPerThread + u < n) s.prefix[tid * kPerThread + u] = m;
    m += own[u];
  }
  __syncthreads();
  // `share` threads, a power of two within a wavefront, split the walk over an entry's bin; the first of them has it.
  int share = 64;
  while (share * n > kSampleThreads && share > 1) share >>= 1;
  const int part = tid & (share - 1);
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    out[u] = {0, 0, 0, -1};
    const int i = tid / share + u * kSampleThreads;
    if (i < n) {
      const Entry e = s.grouped[i];
      const int bin = bin_of(e.word), from = bin == 0 ? 0 : s.cursor[bin - 1], to = s.cursor[bin];
      u64 mass = 0;
      unsigned cnt = 0;
#pragma unroll 4
      for (int j = from + part; j < to; j += share) {
        const Entry o = s.grouped[j];
        if (o.word > e.word) {
          mass += o.mass;
          ++cnt;
        }
      }
      for (int off = 1; off < share; off <<= 1) {
        mass += __shfl_xor(mass, off, 64);
        cnt += __shfl_xor(cnt, off, 64);
      }
      if (part == 0)
        out[u] = {cnt + (whole ? from : s.cnt[bin]), mass + (whole ? s.prefix[from] : s.mass[bin]), e.mass, entry_index(e.word)};
    }
  }
}

// The listed token at position `pos` (by count, or by mass), into s.at; false: not in the list.
__device__ __forceinline__ bool find_listed(SampleLds& s, const Listed (&l)[kPerThread], u64 pos, bool by_mass) {
  if (threadIdx.x == 0) s.found = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPerThread; ++u) {
    const u64 before = by_mass ? l[u].before_mass : l[u].before_cnt, own = by_mass ? l[u].mass : 1;
    if (l[u].token >= 0 && pos >= before && pos - before < own) {
      s.at = l[u];
      s.found = 1;
    }
  }
  __syncthreads();
  const bool found = s.found != 0;
  __syncthreads();  // before another call clears it
  return found;
}

// ------------------------------------------------------------------ radix select

// The histogram of the digit at bits [shift, shift + kDigitBits) of the keys, over the tokens whose key bits
// from `top` on are `prefix`'s; ends with a barrier.
template <typename T>
__device__ __forceinline__ void digit_histogram(SampleLds& s, const T* row, int V, unsigned prefix, int top, int shift, const Weights& ws) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kBins; i += kSampleThreads) s.cnt[i] = 0, s.mass[i] = 0;
  __syncthreads();
  for_row<1>(row, V, [&](T x, int) {
    const unsigned k = Key<T>::of(x);
    if (top < Key<T>::kBits && (k ^ prefix) >> top != 0) return;
    const u64 m = ws(static_cast<float>(x));
    const int bin = k >> shift & (kBins - 1);
    atomicAdd(&s.cnt[bin], 1u);
    if (m != 0) atomicAdd(&s.mass[bin], m);
  });
  __syncthreads();
}

// Inclusive sums over the bins up to this thread's second one, bins first, first + step, ... in this order.
__device__ __forceinline__ void scan_bins(SampleLds& s, int b0, int b1, u64& cnt, u64& mass) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  cnt = (u64)s.cnt[b0] + s.cnt[b1];
  mass = s.mass[b0] + s.mass[b1];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 oc = __shfl_up(cnt, off, 64), om = __shfl_up(mass, off, 64);
    if (lane >= off) cnt += oc, mass += om;
  }
  if (lane == 63) s.wcnt[wave] = (unsigned)cnt, s.wmass[wave] = mass;
  __syncthreads();
  for (int w = 0; w < wave; ++w) cnt += s.wcnt[w], mass += s.wmass[w];
}

struct Place {
  unsigned key;
  u64 before_cnt, before_mass;  // of the tokens with larger keys
};

// The key at position `pos`.
template <typename T>
__device__ __forceinline__ Place locate(SampleLds& s, const T* row, int V, u64 pos, bool by_mass, const Weights& ws) {
  Place p{0, 0, 0};
  const int b0 = kBins - 1 - 2 * threadIdx.x, b1 = b0 - 1;
#pragma unroll 1
  for (int top = Key<T>::kBits; top > 0; top -= kDigitBits) {
    const int shift = max(top - kDigitBits, 0);
    // The last digit reaches above `top` where the key's bits are no multiple of a digit's; the tokens agree there.
    digit_histogram(s, row, V, p.key, top, shift, ws);
    u64 c, m;
    scan_bins(s, b0, b1, c, m);
    for (int e = 1; e >= 0; --e) {
      const int bin = e == 0 ? b0 : b1;
      c -= s.cnt[bin];
      m -= s.mass[bin];
      const u64 before = by_mass ? m : c, own = by_mass ? s.mass[bin] : s.cnt[bin];
      if (pos >= before && pos - before < own) s.bin = bin, s.before_cnt = c, s.before_mass = m;
    }
    __syncthreads();
    p.key = (p.key & ~((unsigned)(kBins - 1) << shift)) | (unsigned)s.bin << shift;
    p.before_cnt += s.before_cnt;
    p.before_mass += s.before_mass;
    pos -= by_mass ? s.before_mass : s.before_cnt;
    __syncthreads();
  }
  return p;
}

// The index of the token of key `key` that `nth` others of that key precede.
template <typename T>
__device__ __forceinline__ int nth_token(SampleLds& s, const T* row, int V, unsigned key, u64 nth) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (V + kSampleThreads - 1) / kSampleThreads * 64, lo = min(wave * per, V), hi = min(lo + per, V);
  unsigned n = 0;
  for (int i = lo + lane; i < hi; i += 64) n += Key<T>::of(row[i]) == key;
#pragma unroll
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

// ------------------------------------------------------------------ the cuts

// The last position by mass that top-p keeps of a top-k of mass `kept`: tokens are kept while the mass before them is
// below p * kept.
__device__ __forceinline__ u64 top_p_position(double p, u64 kept) {
  return static_cast<u64>(fmax(ceil(p * static_cast<double>(kept)), 1.0)) - 1;
}
// The position the uniform number draws of a kept mass.
__device__ __forceinline__ u64 draw_position(double uni, u64 kept) {
  const double at = uni > 0.0 ? uni * static_cast<double>(kept) : 0.0;
  return at < static_cast<double>(kept) ? min(static_cast<u64>(at), kept - 1) : kept - 1;
}

// A bound that at least k (1 to 1024) of the threads' values reach: the k-th largest of them, its key cut to 16 bits.
// Two bits a round, from the top.
__device__ __forceinline__ float kth_of_threads(SampleLds& s, float mine, int k) {
  const unsigned key = key32(mine);
  unsigned bound = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int bit = 30 - 2 * i;
    // How many reach bound + 1, + 2 and + 3 units of these bits, 16 bits each.
    u64 c = 0;
#pragma unroll
    for (unsigned d = 1; d < 4; ++d) c |= (u64)__popcll(__ballot(key >= (bound | d << bit))) << (16 * (d - 1));
    if ((threadIdx.x & 63) == 0) atomicAdd(&s.round[i], c);
    __syncthreads();
    const u64 n = s.round[i];
    const unsigned kk = k, n1 = n & 0xffff, n2 = n >> 16 & 0xffff, n3 = n >> 32;
    bound |= (n3 >= kk ? 3u : n2 >= kk ? 2u : n1 >= kk ? 1u : 0u) << bit;
  }
  return bound <= key32(kNegInf) ? kNegInf : Key<float>::value(bound);
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void coalibi_sample_kernel(SampleArgs a) {
  __shared__ SampleLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, V = a.V;
  const T* const row = static_cast<const T*>(a.logits) + b * a.row_stride;
  const double temp = a.temperature != nullptr ? static_cast<double>(a.temperature[b]) : a.temperature_all;
  const int top_k = a.top_k != nullptr ? a.top_k[b] : a.top_k_all;
  const double top_p = a.top_p != nullptr ? static_cast<double>(a.top_p[b]) : a.top_p_all;
  const double min_p = a.min_p != nullptr ? static_cast<double>(a.min_p[b]) : a.min_p_all;
  const double uni = a.uniforms_f64 ? static_cast<const double*>(a.uniforms)[b]
                                    : static_cast<double>(static_cast<const float*>(a.uniforms)[b]);
  if (tid < 32) s.exp2_table[tid] = kExp2Table[tid] * static_cast<double>(1ull << a.mass_bits);
  if (tid < kRounds) s.round[tid] = 0;
  if (tid < kSums) s.sum[tid] = 0;
  if (tid == 0) s.listed = 0, s.token = V, s.low = key32(__builtin_inff());

  // 1. The largest logit, each thread's smallest, and whether one is NaN (magnitude bits above the infinities').
  float mine = kNegInf, low = __builtin_inff();
  unsigned magnitude = 0;
  for_row<8>(row, V, [&](T x, int) {
    const float f = static_cast<float>(x);
    mine = fmaxf(mine, f);
    low = fminf(low, f);
    magnitude = max(magnitude, __builtin_bit_cast(unsigned, f) & 0x7fffffffu);
  });
  float top = mine;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) s.wcnt[wave] = __builtin_bit_cast(unsigned, top);
  const bool nan = __syncthreads_or(magnitude > 0x7f800000u);
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) top = fmaxf(top, __builtin_bit_cast(float, s.wcnt[w]));
  __syncthreads();
  if (nan || top == kNegInf) {
    if (tid == 0) a.tokens[b] = -1;
    return;
  }
  if (!(temp > 0.0)) {  // 0, negative or NaN: the first of the largest logits
    for_row_if(row, V, [&](T x) { return static_cast<float>(x) == top; }, [&](T, int i) { atomicMin(&s.token, i); });
    __syncthreads();
    if (tid == 0) a.tokens[b] = s.token;
    return;
  }
  unsigned key;
  u64 nth;
  {
    Weights ws;
    ws.top = top;
    ws.top64 = static_cast<double>(top);
    ws.c = 32.0 * 1.4426950408889634074 / temp;
    ws.one = static_cast<double>(1ull << a.mass_bits);
    ws.reach = fmin((a.mass_bits + 2) * static_cast<double>(kLn2) * temp, 0x1p1023);
    ws.table = s.exp2_table;
    const bool cut_k = top_k > 0 && top_k < V, cut_p = top_p < 1.0, cut_m = min_p > 0.0;
    const double min_scaled = min_p * ws.one;
    const u64 one = static_cast<u64>(1) << a.mass_bits;  // the first token's weight

    auto list = [&](int bin, float x, int i) {
      const int at = atomicAdd(&s.listed, 1);
      if (at < kMaxList) s.list[at] = entry_word(bin, x, i);
    };

    // 2. A short list: the first k and what ties with their bound, or (without top-k) the tokens near or above min-p's
    // bound; top-p then also needs the sum of all weights.
    int n = kMaxList + 1;
    u64 all = 0, heavy = 0;  // the weights' sum, and min-p's part of it
    const bool whole = (cut_k && top_k <= kMaxListK) || (!cut_k && cut_m);
    if (whole) {
      float bound;
      if (cut_k) {
        bound = kth_of_threads(s, mine, top_k);
      } else {
        // At the border the weights decide, not this rounding (to them what is 2^-54 below 1 is 1).  Below 2^-126 of the
        // largest no weight is left, and the logarithm stays finite; the product with a temperature of any size is fp64's.
        const float far = fmaxf(-log2f(fmaxf(static_cast<float>(min_p), 0x1p-126f)), 0.f) * (kLn2 * 1.00001f) + 1e-12f;
        bound = static_cast<float>(ws.top64 - static_cast<double>(far) * temp);
        bound -= 1e-6f * (fabsf(top) + fabsf(bound));
        if (top == __builtin_inff()) bound = top;
      }
      // The bins that place_listed groups by: of the distance from the largest, down to the bound.
      const float per_unit = (kBins - 1) / fmaxf(top - bound, 1e-30f);
      auto bin_from = [&](float x) {
        const float d = x == top ? 0.f : (top - x) * per_unit;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
      };
      const bool add_up = !cut_k && cut_p;
      for_row_if(row, V, [&](T x) {
        if (add_up) all += ws(static_cast<float>(x));
        return static_cast<float>(x) >= bound;
      }, [&](T x, int i) { list(bin_from(static_cast<float>(x)), static_cast<float>(x), i); });
      if (add_up) all = block_sum(all, s, 0);
      __syncthreads();
      n = s.listed;
      if (n <= kMaxList && cut_m) {
        for (int i = tid; i < n; i += kSampleThreads) {
          const double w = ws.scaled(entry_logit(s.list[i]));
          if (w >= min_scaled) heavy += Weights::mass(w);
        }
        heavy = block_sum(heavy, s, 1);
      }
    }
    const bool listed = n <= kMaxList;

    // 3. Weights by distance from the largest logit, in equal bins up to the smallest logit or what has no weight; the last
    // bin holds -inf and what lies further.  64 rows of 131072 normal logits, temperature 1.3, top-k
    // 43690 and top-p 0.9: 109 us; with bins up to where weights end, whatever the logits, 429, as the lists do not fit.
    if (!listed) {
      if (low == kNegInf) {  // masked tokens: the smallest of the thread's others
        low = __builtin_inff();
        for_row<8>(row, V, [&](T x, int) {
          const float f = static_cast<float>(x);
          low = fminf(low, f == kNegInf ? low : f);
        });
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) low = fminf(low, __shfl_xor(low, off, 64));
      if (lane == 0) atomicMin(&s.low, key32(low));
      __syncthreads();
      const float span = fminf(static_cast<float>(fmin(ws.reach, 0x1p127)), top - Key<float>::value(s.low));
      const float per_bin = (kBins - 1) * 0.9999f / span;
      auto bin_of = [&](float x) {
        const float d = x == top ? 0.f : (top - x) * per_bin;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
      };
      __syncthreads();
      for (int i = tid; i < kBins; i += kSampleThreads) s.cnt[i] = 0, s.mass[i] = 0;
      if (tid == 0) s.listed = 0;
      __syncthreads();
      heavy = 0;
      for_row<4>(row, V, [&](T x, int) {
        const float f = static_cast<float>(x);
        const double w = ws.scaled(f);
        const u64 m = Weights::mass(w);
        const int bin = bin_of(f);
        if (cut_k) atomicAdd(&s.cnt[bin], 1u);
        if (m != 0) atomicAdd(&s.mass[bin], m);
        if (w >= min_scaled) heavy += m;
      });
      __syncthreads();
      if (cut_m) heavy = block_sum(heavy, s, 2);
      const int b0 = 2 * tid, b1 = b0 + 1;
      const u64 m0 = s.mass[b0], m1 = s.mass[b1];
      const unsigned c0 = s.cnt[b0], c1 = s.cnt[b1];
      u64 c_in, m_in;
      scan_bins(s, b0, b1, c_in, m_in);
      // What lies before this thread's bins takes their place.
      const u64 cb1 = c_in - c1, cb0 = cb1 - c0, mb1 = m_in - m1, mb0 = mb1 - m0;
      __syncthreads();
      s.mass[b0] = mb0;
      s.mass[b1] = mb1;
      s.cnt[b0] = (unsigned)cb0;
      s.cnt[b1] = (unsigned)cb1;
      if (tid == kSampleThreads - 1) s.before_mass = m_in;
      __syncthreads();
      all = s.before_mass;
      __syncthreads();
      // The bins from the one that holds position lo (by mass, or by count) to the one that holds hi; `from` and `to`: the
      // masses before the first and up to the end of the last.
      struct Range {
        int first;
        unsigned more;
      };
      auto range = [&](bool by_mass, u64 lo, u64 hi, u64& from, u64& to) {
        const u64 B0 = by_mass ? mb0 : cb0, B1 = by_mass ? mb1 : cb1, E0 = B0 + (by_mass ? m0 : c0), E1 = B1 + (by_mass ? m1 : c1);
        if (B0 <= lo && lo < E0) s.before_mass = mb0, s.bin = b0;
        if (B1 <= lo && lo < E1) s.before_mass = mb1, s.bin = b1;
        if (B0 <= hi && hi < E0) s.before_cnt = mb0 + m0, s.found = b0;
        if (B1 <= hi && hi < E1) s.before_cnt = mb1 + m1, s.found = b1;
        __syncthreads();
        from = s.before_mass;
        to = s.before_cnt;
        const Range r{s.bin, (unsigned)(s.found - s.bin)};
        __syncthreads();
        return r;
      };
      u64 lo = all, hi = all;  // the kept mass lies in [lo, hi]
      Range at_k{0, 0}, at_p{0, 0};
      if (cut_k) at_k = range(false, top_k - 1, top_k - 1, lo, hi);
      if (cut_p) {
        u64 p_lo, p_hi;
        at_p = range(true, top_p_position(top_p, lo), top_p_position(top_p, hi), p_lo, p_hi);
        lo = min(lo, p_lo);
        hi = min(hi, p_hi);
      }
      if (cut_m) lo = min(lo, max(heavy, one)), hi = min(hi, max(heavy, one));
      lo = max(lo, one);  // the first token is always kept
      hi = max(hi, lo);
      u64 from, to;
      const Range at_u = range(true, draw_position(uni, lo), draw_position(uni, hi), from, to);
      if (!cut_k) at_k = at_u;
      if (!cut_p) at_p = at_u;
      for_row_if(row, V, [&](T x) {
        const int bin = bin_of(static_cast<float>(x));
        return (unsigned)(bin - at_u.first) <= at_u.more || (unsigned)(bin - at_p.first) <= at_p.more ||
               (unsigned)(bin - at_k.first) <= at_k.more;
      }, [&](T x, int i) { list(bin_of(static_cast<float>(x)), static_cast<float>(x), i); });
      __syncthreads();
      n = s.listed;
    }
    heavy = max(heavy, one);

    // The end of the top-k, the end of the top-p and the draw: `end_at(pos, by_mass, end)` finds a position and the mass up
    // to the end of its token; false: it has none.  (Top-p without top-k takes its part of all weights, also where the
    // list holds fewer.)
    auto resolve = [&](u64 cut, auto end_at) {
      u64 end;
      if (cut_k && end_at(top_k - 1, false, end)) cut = end;
      if (cut_p && end_at(top_p_position(top_p, cut_k ? cut : all), true, end)) cut = min(cut, end);
      if (cut_m) cut = min(cut, heavy);
      end_at(draw_position(uni, cut), true, end);
    };
    if (n <= kMaxList) {
      Listed l[kPerThread];
      place_listed(s, n, listed, ws, l);
      resolve(listed ? s.list_mass : all, [&](u64 pos, bool by_mass, u64& end) {
        // Not in the list: past its end, where min-p is the closer cut.
        if (!find_listed(s, l, pos, by_mass)) return false;
        end = s.at.before_mass + s.at.mass;
        return true;
      });
      if (tid == 0) a.tokens[b] = s.at.token;
      return;
    }
    // 4. By radix select.
    resolve(all, [&](u64 pos, bool by_mass, u64& end) {
      const Place p = locate(s, row, V, pos, by_mass, ws);
      const u64 w = ws(Key<T>::value(p.key));
      nth = by_mass ? (pos - p.before_mass) / w : pos - p.before_cnt;  // among the tokens of this key
      end = p.before_mass + (nth + 1) * w;
      key = p.key;
      return true;
    });
  }
  const int token = nth_token(s, row, V, key, nth);
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
