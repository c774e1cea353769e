// Beam search on gfx950: the best continuations over a sequence's beams and the vocabulary, and the paged cache that follows
// them.
//
// Selection: with M_w and S_w a row's largest logit and sum_t exp(x_t - M_w), candidate (w, t) scores
//   score_w + (x_t - M_w) - log S_w.
// Within a row the order is the logits', so that each segment of a row yields its maximum, its sum and its N largest logits in
// one read (its elements stay in registers), and a second launch ranks those of a sequence's beams.  Exponentials are fp32's, each
// within 2^-22 of itself whatever its argument, and their sums fp64's, as scores are until they are written.
//   The N largest of a segment: a bound that N elements reach leaves few above it, which are listed and ranked by counting.  For N up
// to 8 it is the least of N groups of lanes' maxima (about N log N above it), for more the least of the four wavefronts' N / 4-th
// largest lane (about 2 N; but 64 comparisons each).  A logit and its token are one 64-bit key, so that equal logits are in order, too.
//   The ranking takes the lists' first ones first, and stops when every list has come to what is below the N-th best.
//
// Reordering: a group of W beams owns W pages in every column of its block table.  Pages that are full are shared by all that
// descend from them; one in use stays with the first of its heirs, and the others get free pages of its column and copies of
// its rows.  That many are free, as no more than W are in use.  A wavefront works out a column's W beams by itself, a lane
// each, for the tables and again for every copy, so that all is one launch.
//
// Measured in replayed graphs.  Selection, 8 beams of 16 sequences over 131071 bf16 logits, a third of them finished: 22.2 us, of which
// the segments take 14.6 (22.5 MB, which a copy takes 4.6 us for: a segment's loads, its bound, its weights and its list follow one
// another; VALU busy 37 %) and the ranking 7.9, loads and steps of one work-group per sequence in a row.  With exponents rounded as a
// whole, up to 33 weights added in fp32 and rows read from their first 16-byte boundary on, log S was off by 1e-6 and equal rows got
// different sums; it took 18.8, 11.9 and 7.4.  Against that: lists counted by one wavefront 13.8 and 9.4, a bound by counting 64 lanes in
// the segments 14.4, weights against the work-group's maximum 12.9.  4 beams over 50304: 9.5 us.  16 beams of 8 sequences over 50304, 16
// and 32 kept: 23.1 and 37.7 us; 32 of 16 beams over 131072 fp32 34 (groups' bounds for all N and lists one after the other were 1.5,
// 2.4 and 6 times as long).
// Reordering, 4 beams, 24 pools: 4.3 us.  8 beams of 16 sequences, 8 pools of codes and 8 of scales: 11.5 us for 21 MB, which a copy
// takes 4.3 for: 2176 work-groups, of which most find nothing to copy (as many again take 3.5 us more), and three dependent
// reads before a copy's first.  Several pools to a work-group took 12.3, heads over two of them 14.8.
#include <algorithm>

#include "coalibi_common.h"
#include "coalibi_kernels.h"
#include "coalibi_wave.h"

namespace coalibi {

namespace {

constexpr int kSelectThreads = 256;
constexpr int kSelectWaves = kSelectThreads / 64;

// A float as a number of the same order.
__device__ __forceinline__ unsigned ordered(float x) {
  x += 0.f;  // -0 is 0
  const unsigned u = __builtin_bit_cast(unsigned, x);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned k) { return __builtin_bit_cast(float, k ^ ((k >> 31) - 1u | 0x80000000u)); }
// A logit and its token as one number: larger logits first, of equal ones the lower token.  0 is none.
__device__ __forceinline__ u64 logit_key(float x, int token) { return (u64)ordered(x) << 32 | (unsigned)~token; }
__device__ __forceinline__ float key_logit(u64 k) { return unordered((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_token(u64 k) { return (int)~(unsigned)k; }

__device__ __forceinline__ unsigned lane_of(unsigned x, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)x, lane); }
__device__ __forceinline__ u64 lane_of(u64 x, int lane) {
  return (u64)lane_of((unsigned)(x >> 32), lane) << 32 | lane_of((unsigned)x, lane);
}
// Of the largest of groups of a wavefront's numbers, interleaved ones, the least: 2^low groups for `wave`, and 2^max(low - 2, 0)
// for `part`; `top` is the largest of all.  At least 2^low numbers are not below `wave`, and as many of a work-group's not
// below the least of its four wavefronts' `part`.
struct Bounds {
  unsigned wave, part, top;
};
template <int S = 5>
__device__ __forceinline__ void larger_down_to(unsigned& x, int low, int from) {
  if constexpr (S >= 0) {
    if (S >= low && S < from) x = max(x, partner<S>(x));
    larger_down_to<S - 1>(x, low, from);
  }
}
template <int S = 0>
__device__ __forceinline__ void smaller_up_to(unsigned& x, int end) {
  if constexpr (S < 6) {
    if (S < end) x = min(x, partner<S>(x));
    smaller_up_to<S + 1>(x, end);
  }
}
__device__ __forceinline__ Bounds bounds(unsigned x, int low) {
  Bounds r;
  const int fewer = max(low - 2, 0);
  larger_down_to(x, low, 6);
  r.wave = x;
  smaller_up_to(r.wave, low);
  larger_down_to(x, fewer, low);
  r.part = x;
  smaller_up_to(r.part, fewer);
  larger_down_to(x, 0, fewer);
  r.top = x;
  return r;
}

// How many of a wavefront's numbers are larger than a lane's, and the n-th largest (1 <= n <= 64) of them.
__device__ __forceinline__ int larger_lanes(unsigned x) {
  int larger = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) larger += lane_of(x, i) > x ? 1 : 0;
  return larger;
}
__device__ __forceinline__ unsigned nth_of_wave(unsigned x, int larger, int n) {
  u64 is;
  do is = __ballot(larger == --n);  // (equal ones have the first one's count)
  while (is == 0);
  return lane_of(x, __builtin_amdgcn_readfirstlane(__ffsll(is) - 1));
}

// Sums of exp(x) are relative to that of their largest x, m: what is as large weighs 1 exactly, so that a row's only candidate scores
// what its beam does.  Of ordinary m, m log2 e is a whole number and a rest in [-1/2, 1/2], off by 2^-25.
constexpr float kOrdinary = 0x1p20f, kWhole = 0x1.8p23f;
constexpr double kLog2e64 = 0x1.71547652b82fep0;
constexpr float kLog2eRest = (float)(kLog2e64 - (double)kLog2e);
struct Reference {
  float whole, rest;
  __device__ __forceinline__ explicit Reference(float m) : whole(fmaf(m, kLog2e, kWhole) - kWhole), rest(rest_of(m, whole)) {}
  static __device__ __forceinline__ float rest_of(float x, float k) { return fmaf(x, kLog2eRest, fmaf(x, kLog2e, -k)); }
};
// A sum against `from` as one against `to`, which is not less.
__device__ __forceinline__ double rescaled(double sum, float from, float to) {
  if (from == to) return sum;  // (infinities, too)
  if (fabsf(from) < kOrdinary && fabsf(to) < kOrdinary) {
    const Reference a(from), b(to);
    return ldexp(sum * exp2((double)a.rest - (double)b.rest), (int)(a.whole - b.whole));
  }
  return sum * exp2(((double)from - (double)to) * kLog2e64);
}
// exp(x - m) for an ordinary m and x <= m, or NaN.  x log2 e is split as m's is, so that whatever x is the exponent is off by 3 * 2^-25,
// the weight by 2^-24 of itself, and its power by 2^-23 (one step of v_exp_f32): 2^-22.  (A product that is rounded as a whole, 17 for
// a logit that 2^20 of make as heavy as the largest, is off by 2^-20.)  What is below 2^-126 may come to 0.
struct Weights {
  float least, magic, rest;
  __device__ __forceinline__ explicit Weights(float m) : least(m - 128.f) {
    const Reference r(m);
    magic = kWhole - r.whole;
    rest = r.rest;
  }
  __device__ __forceinline__ double operator()(float x) const {
    x = x < least ? least : x;
    const float t = fmaf(x, kLog2e, magic);  // the whole numbers' difference in its last bits: t lies in [2^23, 2^24)
    const float d = Reference::rest_of(x, t - magic) - rest;
    return (double)ldexpf(fast_exp2(d), __builtin_bit_cast(int, t) - __builtin_bit_cast(int, kWhole));
  }
};

constexpr int kListed = 256;  // keys of a wavefront's list, which are ranked by counting

// The lanes' place behind n others, of those for which `is`, and how many they are.
__device__ __forceinline__ int place_of(u64 is) { return __builtin_amdgcn_mbcnt_hi((unsigned)(is >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)is, 0)); }

// C: 16-byte chunks of a segment per thread.  A row's chunks begin with its first token wherever it lies (loads need only an element's
// alignment), so that equal rows are added in the same order and get the same bits: their scores tie.  The tokens behind the last whole
// chunk go with the last segment, one per thread.
template <typename T, int C>
__global__ __launch_bounds__(kSelectThreads) void coalibi_select_rows_kernel(SelectArgs a) {
  constexpr int PER = 16 / sizeof(T), E = C * PER + 1;
  typedef T chunk_t __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
  __shared__ u64 list[kSelectWaves][kListed];
  __shared__ int listed[kSelectWaves], count[kSelectWaves][64];
  __shared__ u64 wnext[kSelectWaves];
  __shared__ unsigned wcut[kSelectWaves], wpart[kSelectWaves];
  __shared__ float wmax[kSelectWaves];
  __shared__ double wsum[kSelectWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), seg = blockIdx.x;
  const long long row = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  if (row >= (long long)a.B * a.W) return;
  if (a.finished != nullptr && a.finished[row] != 0) return;
  const int b = (int)(row / a.W), w = (int)(row - (long long)b * a.W);
  const T* const x = static_cast<const T*>(a.logits) + (size_t)b * a.batch_stride + (size_t)w * a.beam_stride;
  const int chunks = a.V / PER, tail = a.V - chunks * PER;

  const bool ragged = (seg + 1) * (C * kSelectThreads) > chunks;  // not every thread has all of its chunks
  float v[E];
  int where = -1;  // the single element's token
  if (seg == a.segments - 1 && tid < tail) where = a.V - tail + tid;
  v[E - 1] = where >= 0 ? static_cast<float>(x[where]) : kNegInf;
  const int first = seg * (C * kSelectThreads) + tid;  // the thread's first chunk
  if (chunks > 0) {
    chunk_t y[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
      y[c] = *reinterpret_cast<const chunk_t*>(x + (size_t)min(first + c * kSelectThreads, chunks - 1) * PER);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < PER; ++e) v[c * PER + e] = static_cast<float>(y[c][e]);
    if (ragged) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (first + c * kSelectThreads >= chunks) {
#pragma unroll
          for (int e = 0; e < PER; ++e) v[c * PER + e] = kNegInf;
        }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E - 1; ++e) v[e] = kNegInf;
  }
  auto token = [&](int e) { return e == E - 1 ? where : (first + e / PER * kSelectThreads) * PER + e % PER; };

  // The segment's maximum, and a bound that its N-th largest logit is not below.
  float top = v[E - 1];
#pragma unroll
  for (int e = 0; e < E - 1; ++e) top = fmaxf(top, v[e]);
  // A bound from all four wavefronts, and one from each alone (where the others may have few elements).
  const unsigned none = ordered(kNegInf), key = ordered(fmaxf(top, kNegInf));
  const int quarter = (a.N + kSelectWaves - 1) / kSelectWaves;
  unsigned most = 0, fourth = none, single = none;
  if (a.N <= 8) {
    const Bounds x = bounds(key, a.N > 4 ? 3 : a.N > 2 ? 2 : a.N - 1);
    most = x.top;
    fourth = x.part;
    single = x.wave;
  } else {
    const int larger = larger_lanes(key);
    most = nth_of_wave(key, larger, 1);
    fourth = nth_of_wave(key, larger, quarter);
    if (ragged) single = nth_of_wave(key, larger, a.N);
  }
  // The weights' sum, against the wavefront's maximum (the others' are on their way): NaN where there is a NaN.
  const float wm = unordered(most);
  double sum = 0.0;
  if (fabsf(wm) < kOrdinary) {
    const Weights of(wm);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += of(v[e]);
  } else if (fabsf(wm) < __builtin_inff()) {
    const Weights of(0.f);  // (exact for every logit that counts)
#pragma unroll
    for (int e = 0; e < E; ++e) sum += of(v[e] - wm);
  } else {
    float n = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) n += v[e] != v[e] ? v[e] : v[e] == __builtin_inff() ? 1.f : 0.f;
    sum = n;
  }
  if (lane == 0) {
    wcut[wave] = single;
    wpart[wave] = fourth;
    wmax[wave] = wm;
  }
  __syncthreads();
  unsigned least = 0, part_least = ~0u;
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    m = fmaxf(m, wmax[i]);
    least = max(least, wcut[i]);
    part_least = min(part_least, wpart[i]);
  }
  least = max(least, part_least);
  const float low = unordered(least);
  int mine = 0;
  if (__any(top >= low)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!__any(v[e] >= low)) continue;
      const bool in = v[e] >= low && v[e] > kNegInf;
      const u64 is = __ballot(in);
      const int p = mine + place_of(is);
      if (in && p < kListed) list[wave][p] = logit_key(v[e], token(e));
      mine += __popcll(is);
    }
  }
  if (lane == 0) listed[wave] = mine;
  const double total = rescaled(wave_sum(sum), wm, m);
  if (lane == 0) wsum[wave] = total;
  __syncthreads();
  const size_t part = (size_t)row * a.segments + seg;
  const double all = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
  const bool nan = all != all;
  if (tid == 0) {
    a.pmax[part] = nan ? __builtin_nanf("") : m;
    a.psum[part] = all;
  }
  if (nan) return;
  u64* const out = a.pkey + part * a.N;
  int c = 0;
  bool fits = true;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    c += listed[i];
    fits = fits && listed[i] <= kListed;
  }
  if (c <= 64) {  // one each for the lanes; every wavefront counts its share of the larger ones
    int at = lane, from = 0;
#pragma unroll
    for (int i = 0; i < kSelectWaves - 1; ++i)
      if (from == i && at >= listed[i]) {
        at -= listed[i];
        ++from;
      }
    const u64 k = lane < c ? list[from][at] : 0;
    int larger = 0;
    for (int j = wave; j < c; j += kSelectWaves) larger += lane_of(k, j) > k ? 1 : 0;
    count[wave][lane] = larger;
    __syncthreads();
    if (wave == 0) {
      int rank = 0;
#pragma unroll
      for (int i = 0; i < kSelectWaves; ++i) rank += count[i][lane];
      if (lane >= c) rank = lane;
      if (rank < a.N) out[rank] = k;
    }
  } else if (fits) {
    for (int i = lane; i < mine; i += 64) {
      const u64 k = list[wave][i];
      int rank = 0;
      for (int w = 0; w < kSelectWaves; ++w)
        for (int j = 0; j < listed[w]; ++j) rank += list[w][j] > k ? 1 : 0;
      if (rank < a.N) out[rank] = k;
    }
    for (int i = c + tid; i < a.N; i += kSelectThreads) out[i] = 0;
  } else {
    // Too many to list (threads with many of the largest): the next one, N times.
    u64 last = ~0ull;
    for (int n = 0; n < a.N; ++n) {
      u64 k = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[e] > kNegInf) {
          const u64 y = logit_key(v[e], token(e));
          if (y < last && y > k) k = y;
        }
      k = wave_max(k);
      __syncthreads();
      if (lane == 0) wnext[wave] = k;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kSelectWaves; ++i) k = wnext[i] > k ? wnext[i] : k;
      if (tid == 0) out[n] = k;
      last = k;
    }
  }
}

// A score as a number of the same order, above 0.
__device__ __forceinline__ u64 score_key(double x) {
  x += 0.0;
  const u64 u = __builtin_bit_cast(u64, x);
  return u ^ ((u64)((long long)u >> 63) | 1ull << 63);
}
__device__ __forceinline__ double key_score(u64 k) {
  const u64 u = k ^ ((k >> 63) - 1 | 1ull << 63);
  return __builtin_bit_cast(double, u);
}

constexpr int kRound = 8;  // candidates of a thread and round

// The N best of a sequence's candidates, kRound per thread at a time, with the N best so far.  The list has room for all of a
// round's, and few are on it, as in the segments.
__global__ __launch_bounds__(kSelectThreads) void coalibi_select_beams_kernel(SelectArgs a) {
  constexpr int kMost = 64 * (kRound + 1);
  // Candidates: keys of score and logit, and the beam.  Equal scores go by beam, then by the logit's key.
  __shared__ double sbase[kMaxBeams];  // score - log S, or NaN for a beam without candidates
  __shared__ float smax[kMaxBeams];
  __shared__ bool sdone[kMaxBeams];
  __shared__ u64 lscore[kSelectWaves][kMost], llogit[kSelectWaves][kMost], kscore[kMaxBeams], klogit[kMaxBeams];
  __shared__ int lbeam[kSelectWaves][kMost], kbeam[kMaxBeams];
  __shared__ unsigned wcut[kSelectWaves], wpart[kSelectWaves], wbest[kSelectWaves];
  __shared__ int listed[kSelectWaves], count[kSelectWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x;
  const long long row0 = (long long)b * a.W;
  // Candidate i is the i / lists-th of list i % lists (a beam's segment), so that each thread has lists' first ones to begin with.
  const int lists = a.W * a.segments, total = lists * a.N;
  const u64* const from = a.pkey + (size_t)row0 * a.segments * a.N;
  const int by_n = (unsigned)kSelectThreads / (unsigned)lists, by_list = kSelectThreads - by_n * lists;
  struct Place {
    int n, list;
  };
  auto place_at = [&](int first) {
    const unsigned i = (unsigned)(first + tid), n = i / (unsigned)lists;
    return Place{(int)n, (int)(i - n * (unsigned)lists)};
  };
  auto next = [&](Place& p) {  // kSelectThreads later
    p.n += by_n;
    p.list += by_list;
    if (p.list >= lists) {
      p.list -= lists;
      ++p.n;
    }
  };
  u64 keys[kRound];  // of the first round, on their way meanwhile
  auto load_keys = [&](int first) {
    Place p = place_at(first);
#pragma unroll
    for (int r = 0; r < kRound; ++r, next(p)) keys[r] = from[(size_t)p.list * a.N + min(p.n, a.N - 1)];
  };
  load_keys(0);
  const float per_segment = 1.f / a.segments;  // (a quotient below 64, half a segment from the next: no rounding reaches it)
  for (int w = wave; w < a.W; w += kSelectWaves) {
    const long long row = row0 + w;
    const float score = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    double base = done ? (double)score : __builtin_nan("");
    float m = 0.f;
    if (!done) {
      const float* const pm = a.pmax + row * a.segments;
      const double* const ps = a.psum + row * a.segments;
      const float m0 = lane < a.segments ? pm[lane] : kNegInf;
      const double s0 = lane < a.segments ? ps[lane] : 0.0;
      bool nan = m0 != m0;
      m = fmaxf(m0, kNegInf);
      for (int s = lane + 64; s < a.segments; s += 64) {
        nan |= pm[s] != pm[s];
        m = fmaxf(m, pm[s]);
      }
      m = wave_max(m);
      double sum = rescaled(s0, m0, m);
      for (int s = lane + 64; s < a.segments; s += 64) sum += rescaled(ps[s], pm[s], m);
      sum = wave_sum(sum);
      if (!__any(nan) && m > kNegInf) base = (double)score - log(sum);
    }
    if (lane == 0) {
      sbase[w] = score > kNegInf && score < __builtin_inff() ? base : __builtin_nan("");
      smax[w] = m;
      sdone[w] = done;
    }
  }
  if (tid < a.N) {
    kscore[tid] = klogit[tid] = 0;
    kbeam[tid] = 0;
  }
  __syncthreads();
  for (int first = 0; first < total; first += kRound * kSelectThreads) {
    u64 score[kRound + 1], logit[kRound + 1];
    int beam[kRound + 1];
    Place p = place_at(first);
#pragma unroll
    for (int r = 0; r < kRound; ++r, next(p)) {
      score[r] = logit[r] = 0;
      beam[r] = 0;
      if (p.n < a.N) {
        const int w = (int)(((float)p.list + 0.5f) * per_segment);
        const double base = sbase[w];
        const bool done = sdone[w];
        u64 k = keys[r];
        const float x = key_logit(k), m = smax[w];
        if (done) k = p.n == 0 && p.list == w * a.segments ? logit_key(0.f, a.end_token) : 0;
        // Of +inf logits all weigh 1, and every other one nothing.
        if (base == base && k != 0 && (done || x == m || m < __builtin_inff())) {
          score[r] = score_key(done || x == m ? base : base + ((double)x - (double)m));
          logit[r] = k;
          beam[r] = w;
        }
      }
    }
    score[kRound] = tid < a.N ? kscore[tid] : 0;
    logit[kRound] = tid < a.N ? klogit[tid] : 0;
    beam[kRound] = tid < a.N ? kbeam[tid] : 0;
    if (first + kRound * kSelectThreads < total) load_keys(first + kRound * kSelectThreads);
    u64 best = 0;
#pragma unroll
    for (int r = 0; r < kRound; ++r) best = score[r] > best ? score[r] : best;
    // No more than the N-th largest candidate: the N-th of those before; a wavefront's N-th largest lane, by the scores' first halves;
    // and the least of four wavefronts' N / 4-th.
    const unsigned lead = (unsigned)(best >> 32);
    const int larger = larger_lanes(lead);
    const unsigned cut = nth_of_wave(lead, larger, a.N), part = nth_of_wave(lead, larger, (a.N + kSelectWaves - 1) / kSelectWaves);
    if (lane == 0) {
      wcut[wave] = cut;
      wpart[wave] = part;
      wbest[wave] = 0;
    }
    u64 least = max(kscore[a.N - 1], 1ull);
    if (first > 0 && __any(best >= least) && lane == 0) wbest[wave] = 1;
    __syncthreads();
    // A round in which every list is below the N-th already: so is what follows of each.
    if (first > 0 && lists <= kRound * kSelectThreads && (wbest[0] | wbest[1] | wbest[2] | wbest[3]) == 0) break;
    unsigned part_least = ~0u;
#pragma unroll
    for (int i = 0; i < kSelectWaves; ++i) {
      least = max(least, (u64)wcut[i] << 32);
      part_least = min(part_least, wpart[i]);
    }
    least = max(least, (u64)part_least << 32);
    int mine = 0;
#pragma unroll
    for (int r = 0; r <= kRound; ++r) {
      const u64 is = __ballot(score[r] >= least);
      if (is == 0) continue;
      const int p = mine + place_of(is);
      if (score[r] >= least) {
        lscore[wave][p] = score[r];
        llogit[wave][p] = logit[r];
        lbeam[wave][p] = beam[r];
      }
      mine += __popcll(is);
    }
    if (lane == 0) listed[wave] = mine;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) n += listed[w];
    if (tid < a.N && tid >= n) {
      kscore[tid] = klogit[tid] = 0;
      kbeam[tid] = 0;
    }
    if (n <= 64) {  // one each for the lanes; every wavefront counts its share of the larger ones
      int at = lane, from = 0;
#pragma unroll
      for (int i = 0; i < kSelectWaves - 1; ++i)
        if (from == i && at >= listed[i]) {
          at -= listed[i];
          ++from;
        }
      const bool is = lane < n;
      const u64 x = is ? lscore[from][at] : 0, xl = is ? llogit[from][at] : 0;
      const int xb = is ? lbeam[from][at] : 0;
      int larger = 0;
      for (int j = wave; j < n; j += kSelectWaves) {
        const u64 y = lane_of(x, j);
        const int yb = __builtin_amdgcn_readlane(xb, j);
        larger += y > x || (y == x && (yb < xb || (yb == xb && lane_of(xl, j) > xl))) ? 1 : 0;
      }
      count[wave][lane] = larger;
      __syncthreads();
      if (wave == 0) {
        int rank = 0;
#pragma unroll
        for (int i = 0; i < kSelectWaves; ++i) rank += count[i][lane];
        if (is && rank < a.N) {
          kscore[rank] = x;
          klogit[rank] = xl;
          kbeam[rank] = xb;
        }
      }
    } else {
      for (int i = lane; i < mine; i += 64) {
        const u64 x = lscore[wave][i], xl = llogit[wave][i];
        const int xb = lbeam[wave][i];
        int rank = 0;
        for (int w = 0; w < kSelectWaves; ++w)
          for (int j = 0; j < listed[w]; ++j) {
            const u64 y = lscore[w][j];
            if (y > x)
              ++rank;
            else if (y == x)
              rank += lbeam[w][j] < xb || (lbeam[w][j] == xb && llogit[w][j] > xl) ? 1 : 0;
          }
        if (rank < a.N) {
          kscore[rank] = x;
          klogit[rank] = xl;
          kbeam[rank] = xb;
        }
      }
    }
    __syncthreads();
  }
  if (tid < a.N) {
    const u64 x = kscore[tid];
    const size_t o = (size_t)b * a.N + tid;
    a.out_scores[o] = x == 0 ? kNegInf : (float)key_score(x);
    a.out_parents[o] = kbeam[tid];
    a.out_tokens[o] = x == 0 ? -1 : key_token(klogit[tid]);
  }
}

// What becomes of a group's pages in one column; lane i is beam i.
struct Column {
  int from, to;  // the parent's page, the beam's
  int rows;      // filled rows of it, all of which `to` has to get where it is another page
  int len;
  bool copies;
};
// A group's parents and its beams' new lengths, a lane each.
struct Heirs {
  int parent, len;
};
__device__ __forceinline__ Heirs heirs(const ReorderArgs& a, int g, int lane) {
  const size_t mine = (size_t)g * a.W + (lane < a.W ? lane : 0);
  const int parent = min(max(a.parents[mine], 0), a.W - 1);
  return {parent, __shfl(a.lens[mine], parent, 64)};
}
__device__ __forceinline__ Column column(const ReorderArgs& a, const Heirs& x, int g, int j, int lane, int* free_pages) {
  const bool is = lane < a.W;
  const size_t mine = (size_t)g * a.W + (is ? lane : 0);
  Column c;
  c.len = x.len;
  c.from = __shfl(a.table[mine * a.J + j], x.parent, 64);
  const int home = a.pages[mine * a.J + j];
  c.rows = (int)min(max((long long)c.len - (long long)j * a.page, 0ll), (long long)a.page);
  const bool full = is && c.rows == a.page, part = is && c.rows > 0 && !full;
  const unsigned long long fulls = __ballot(full), parts = __ballot(part);
  bool taken = false;
  for (int k = 0; k < a.W; ++k) {
    const bool same = __shfl(c.from, k, 64) == c.from;
    taken |= same && ((fulls >> k & 1) || ((parts >> k & 1) && k < lane));
  }
  const bool keeps = full || (part && !taken);
  const unsigned long long keep = __ballot(keeps);
  bool used = false;
  for (int k = 0; k < a.W; ++k) {
    const int page = __shfl(c.from, k, 64);
    used |= (keep >> k & 1) && page == home;
  }
  const unsigned long long free = __ballot(is && !used), needs = __ballot(is && !keeps), below = (1ull << lane) - 1;
  if (is && !used) free_pages[__popcll(free & below)] = home;
  wait_lds();  // a wavefront's LDS operations complete in order
  const int place = __popcll(needs & below);
  c.to = keeps ? c.from : place < __popcll(free) ? free_pages[place] : home;
  c.copies = part && !keeps;
  return c;
}

constexpr int kReorderThreads = 256;

// The first bytes of each head of a page, eight pieces a thread on their way at once.
template <typename V>
__device__ __forceinline__ void copy_heads(char* dst, const char* src, int bytes, int heads, long long stride, int tid) {
  constexpr int N = 8;
  const unsigned n = (unsigned)bytes / (unsigned)sizeof(V), all = n * (unsigned)heads;
  for (unsigned i = tid; i < all; i += kReorderThreads * N) {
    V x[N];
    long long at[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const unsigned j = min(i + kReorderThreads * e, all - 1), h = j / n;
      at[e] = (long long)h * stride + (long long)(j - h * n) * (int)sizeof(V);
      x[e] = *reinterpret_cast<const V*>(src + at[e]);
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (i + kReorderThreads * e < all) *reinterpret_cast<V*>(dst + at[e]) = x[e];
  }
}

__global__ __launch_bounds__(kReorderThreads) void coalibi_reorder_kernel(ReorderArgs a) {
  __shared__ int sfree[kReorderThreads / 64][64];
  __shared__ int smove[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int beams = a.B * a.W;
  if (blockIdx.y == (unsigned)a.pools) {  // the tables: a wavefront per group and column
    const long long columns = (long long)a.B * a.J;
    for (long long at = (long long)blockIdx.x * (kReorderThreads / 64) + wave; at < columns;
         at += (long long)gridDim.x * (kReorderThreads / 64)) {
      const int g = (int)(at / a.J), j = (int)(at - (long long)g * a.J);
      const Column c = column(a, heirs(a, g, lane), g, j, lane, sfree[wave]);
      if (lane < a.W) {
        a.out_table[((size_t)g * a.W + lane) * a.J + j] = c.to;
        if (j == 0) a.out_lens[(size_t)g * a.W + lane] = c.len;
      }
    }
    return;
  }
  // A beam's copies in one pool.
  const PoolDesc& p = a.pool[blockIdx.y];
  for (int i = blockIdx.x; i < beams; i += gridDim.x) {
    const int g = i / a.W, w = i - g * a.W;
    if (wave == 0) {
      const Heirs x = heirs(a, g, lane);
      const int len = __shfl(x.len, w, 64), j = len >> a.page_shift;
      int from = -1, to = -1, rows = 0;
      if (len > 0 && j < a.J && (len & (a.page - 1)) != 0) {  // there is a page in use
        const Column c = column(a, x, g, j, lane, sfree[0]);
        rows = __ballot(c.copies) >> w & 1 ? __shfl(c.rows, w, 64) : 0;
        from = __shfl(c.from, w, 64);
        to = __shfl(c.to, w, 64);
      }
      if (lane == 0) {
        const bool in = from >= 0 && from < a.num_pages && to >= 0 && to < a.num_pages;
        smove[0] = from;
        smove[1] = to;
        smove[2] = in ? rows : 0;
      }
    }
    __syncthreads();
    const int from = smove[0], to = smove[1], rows = smove[2];
    __syncthreads();
    if (rows == 0) continue;
    const int bytes = (int)(((long long)rows * p.entries + a.page - 1) / a.page) * p.entry_bytes;  // of each head
    const char* const src = p.p + (size_t)from * p.page_stride;
    char* const dst = p.p + (size_t)to * p.page_stride;
    if (p.wide)
      copy_heads<u32x4>(dst, src, bytes, p.heads, p.head_stride, tid);
    else
      copy_heads<unsigned>(dst, src, bytes, p.heads, p.head_stride, tid);
  }
}

}  // namespace

template <typename T>
hipError_t launch_select(const SelectArgs& a, hipStream_t stream) {
  const long long rows = (long long)a.B * a.W;
  const unsigned y = static_cast<unsigned>(std::min<long long>(rows, 32768));
  const dim3 grid(static_cast<unsigned>(a.segments), y, static_cast<unsigned>((rows + y - 1) / y));
  switch (a.chunks) {
    case 1: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 1>), grid, dim3(kSelectThreads), 0, stream, a); break;
    case 2: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 2>), grid, dim3(kSelectThreads), 0, stream, a); break;
    default: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 4>), grid, dim3(kSelectThreads), 0, stream, a); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(coalibi_select_beams_kernel, dim3(static_cast<unsigned>(a.B)), dim3(kSelectThreads), 0, stream, a);
  return hipGetLastError();
}
template hipError_t launch_select<_Float16>(const SelectArgs&, hipStream_t);
template hipError_t launch_select<__bf16>(const SelectArgs&, hipStream_t);
template hipError_t launch_select<float>(const SelectArgs&, hipStream_t);

hipError_t launch_reorder(const ReorderArgs& a, hipStream_t stream) {
  const long long columns = (long long)a.B * a.J, beams = (long long)a.B * a.W;
  const long long x = std::max(a.pools > 0 ? beams : 1, a.tables ? (columns + 3) / 4 : 1);
  const dim3 grid(static_cast<unsigned>(std::min<long long>(x, 65535)), static_cast<unsigned>(a.pools + (a.tables ? 1 : 0)));
  hipLaunchKernelGGL(coalibi_reorder_kernel, grid, dim3(kReorderThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace coalibi
