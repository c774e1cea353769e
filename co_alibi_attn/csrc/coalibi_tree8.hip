// Co-ALiBi attention of a step's new tokens over a key / value cache held in 8 bits, and each other, on gfx950.
//
// The definition is the tree decode's (coalibi_tree.hip) with cached keys ks * kc and values vs * vc: codes kc, vc (e4m3 or
// int8) and a scale for each kv head's block of 16 rows.  A code is a 16-bit type's own value, so the codes go into the
// products as they are and the scales outside of them:
//   t_j = sm_scale*log2(e) * ks * (q.kc_j),   a_j = t_j - slope*log2(e) * z_j,   a'_j = a_j + log2 vs,
//   O   = sum_j 2^(a'_j - m) vc_j / l,   l = sum_j 2^(a'_j - m) / vs,   LSE = (m + log2 l) * ln 2.
// The lane of a score holds the 16 keys of a block, so ks is a factor of its scores' one multiplication, log2 vs a part of
// the one term that all of its exponents subtract, and 1 / vs one multiplication for their sum.  (With fp16 weights the codes take the
// powers of two of vs instead, which leaves the weights their bits: no slower.)
//
// A wavefront takes 32 query rows over a run of 32-key tiles, newest first, by itself: S^T = K Q^T and O^T += V^T P^T on MFMA,
// the operands straight from memory into registers.
//   K: a lane reads 16 bytes of its key's row, the codes of two k16 steps; Q is laid out to match.
//   V: a lane reads D / 32 consecutive codes of each of its half's 16 keys; output row R of tile j is d = (D / 32) * R + j, so
// they are one element of each tile's operand.  Two keys' codes are interleaved by byte permutes and converted as pairs.
// There are no barriers and no LDS in the loop.  The four wavefronts of a work-group take four runs of a split's tiles and are
// joined at its end, each one's maximum shifted by the sigmas of the keys after it, as splits are in the merge.
//
// What bounds it, by replayed graphs and counters (D 128; both kernels, of which the merge takes 4.7 us, for drafts 9.4):
//   one token for each of 32 sequences of up to 8192 rows (32 / 8 heads, bf16, e4m3): 63 us; 259 of 301 MB are read (values of far
//     keys are not) at 5.0 TB/s, VALU busy 39 %, MFMA 11 %;
//   24 drafts for each of 16 (int8): 82 us; VALU busy 50 %, MFMA 11 %: int8 has no conversion to bf16 (three instructions for two
//     codes, e4m3 has one), and about 12 of them go with each score;
//   7 drafts over 131072 rows (fp16, e4m3): 57 us; 233 MB at 5.1 TB/s;
//   one token over 500 rows of 12 heads (bf16 D 64): 9.5 us in one work-group a head, the latency of its tiles in a row;
//   8 tokens for each of 4 over 8192 rows (8 heads, fp32, e4m3): 62 us: products of 32 rows for 8, at a 16th of bf16's rate.
// Taken step by step for the 32 sequences, the drafts and the long one: keys and values loaded where they are used 71, 115 and 64
// us; keys a tile ahead, values while a tile is weighed, their product with the weights a tile late 67, 117 and 57; plans by the
// batch's own lengths, two rounds of work-groups where several row blocks share keys: drafts 86; splits by kv head, the
// flattest first 64, 84 and 56; a plan's lengths read once: drafts 82.  Keys two tiles ahead: 63 in place of 64, but D 256 spills.
#include <algorithm>
#include <type_traits>

#include "coalibi_tree.h"

namespace coalibi {

namespace {

constexpr int kTree8Waves = 4;
constexpr int kTree8Threads = 64 * kTree8Waves;

typedef unsigned short u16;

// Byte N of x, an int8, as a float: one conversion that picks the byte.  (A shift and a cast took two instructions for odd bytes.)
template <int N>
__device__ __forceinline__ float signed_byte(unsigned x) {
  return static_cast<float>((int)__builtin_amdgcn_sbfe((int)x, 8 * N, 8));
}

// Two floats of at most 8 significant bits as two bfloat16.
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060302u);
}
// A power of two 2^e that fp16's operands of V are taken by: exact for all codes from 2^-15 to 2^7 (e4m3: 2^-9 to 448), or from 2^-24
// to 2^5 (int8: 1152 * 2^5 is a number of fp16, too).  The other types' weights have the range that scales need.
struct Times1 {
  __device__ __forceinline__ explicit Times1(int = 0) {}
};
template <typename F>
struct TimesPower {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  float f;         // 2^e
  f16x2 h, minus;  // int8: 2^e and -1152 * 2^e twice
  __device__ __forceinline__ explicit TimesPower(int e) : f(ldexpf(1.f, e)) {
    if constexpr (__is_same(F, I8)) {
      const _Float16 x = static_cast<_Float16>(f);
      h = f16x2{x, x};
      minus = h * f16x2{(_Float16)-1152.0f, (_Float16)-1152.0f};
    }
  }
};
// Pair HI (bytes 0 and 1, or 2 and 3) of the codes in x, as the bits of two 16-bit T.
template <typename T, typename F, bool HI, typename P>
__device__ __forceinline__ unsigned code_pair(unsigned x, const P& by) {
  if constexpr (__is_same(F, E4M3) && __is_same(T, __bf16)) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, HI));
  } else if constexpr (__is_same(F, E4M3)) {
    float f = 1.0f;
    if constexpr (!__is_same(P, Times1)) f = by.f;
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, f, HI));
  } else if constexpr (__is_same(T, _Float16)) {
    // The byte plus 128 in the last bits of 1024: exact, and so is the difference, and its product with the power of two.
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const unsigned h = __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u, HI ? 0x05030402u : 0x05010400u);
    if constexpr (__is_same(P, Times1))
      return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, h) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f});
    else
      return __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, h), by.h, by.minus));
  } else {
    return pack_bf16(signed_byte<HI ? 2 : 0>(x), signed_byte<HI ? 3 : 1>(x));
  }
}
// Byte N of x, a code, as a float.
template <typename F, int N>
__device__ __forceinline__ float code_float(unsigned x) {
  if constexpr (__is_same(F, E4M3)) return __builtin_amdgcn_cvt_f32_fp8((int)x, N);
  return signed_byte<N>(x);
}
// Eight codes, four of lo and four of hi, as a product's operand.
template <typename T, typename F>
__device__ __forceinline__ typename Mfma<T>::vec8 code_vec8(unsigned lo, unsigned hi) {
  if constexpr (sizeof(T) == 2)
    return __builtin_bit_cast(typename Mfma<T>::vec8, u32x4{code_pair<T, F, false>(lo, Times1()), code_pair<T, F, true>(lo, Times1()),
                                                            code_pair<T, F, false>(hi, Times1()), code_pair<T, F, true>(hi, Times1())});
  else
    return f32x8{code_float<F, 0>(lo), code_float<F, 1>(lo), code_float<F, 2>(lo), code_float<F, 3>(lo),
                 code_float<F, 0>(hi), code_float<F, 1>(hi), code_float<F, 2>(hi), code_float<F, 3>(hi)};
}
// Byte N of eight words as an operand.  Of two words at a time, the byte of both as a pair.
template <typename T, typename F, int N, typename P>
__device__ __forceinline__ typename Mfma<T>::vec8 byte_vec8(const unsigned (&w)[8], const P& by) {
  if constexpr (sizeof(T) == 4) {
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = code_float<F, N>(w[e]);
    return x;
  } else {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (__is_same(F, I8) && __is_same(T, __bf16))
        x[e] = pack_bf16(signed_byte<N>(w[2 * e]), signed_byte<N>(w[2 * e + 1]));
      else  // (the permute serves the next byte, too)
        x[e] = code_pair<T, F, (N & 1) != 0>(__builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], N & 2 ? 0x07030602u : 0x05010400u), by);
    }
    return __builtin_bit_cast(typename Mfma<T>::vec8, x);
  }
}

// D / 32 consecutive codes, at least one.
template <int DT>
struct Run {
  static constexpr int W = DT > 4 ? DT / 4 : 1;
  unsigned w[W];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (DT == 8) {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      w[0] = x[0];
      w[1] = x[1];
    } else if constexpr (DT == 4) {
      w[0] = *reinterpret_cast<const unsigned*>(p);
    } else if constexpr (DT == 2) {
      w[0] = *reinterpret_cast<const u16*>(p);
    } else {
      w[0] = *reinterpret_cast<const unsigned char*>(p);
    }
  }
};

// A tile's keys as a lane holds them, and its half's scales.
template <int D>
struct Keys8 {
  static constexpr int KL = D < 32 ? 1 : D / 32;  // 16-byte pieces of a key (D 16: 8 bytes)
  u32x4 k[KL];
  float ks, vs;
};

template <typename T, int D>
struct Tree8Cfg {
  static constexpr int KS = D / 16;
  static constexpr int DT = D < 32 ? 1 : D / 32;
  static constexpr int LDO = D + 4;  // a wavefront's O rows in LDS, 16 bytes apart from a power of two
  static constexpr int LDS_BYTES = kTree8Waves * 32 * LDO * 4;
  static constexpr int WGS_PER_CU = D * sizeof(T) <= 256 ? 2 : 1;
};

// Whether a scale is one that the formulas hold for: from the smallest to the largest (a NaN is not).
__device__ __forceinline__ bool scale_ok(float s) { return s >= kScaleLeast && s <= kScaleMost; }

// As plan_item, but by kv head, the last head first: its slopes are the flattest where their number is a power of two, and the tiles
// of flat heads, of which few are left out, take the longest.
__device__ __forceinline__ TreeItem head_item(const TreeArgs& a, int cps, int id, int lane, int first) {
  auto splits = [&](int b0) {
    const int chunks = lane_chunks(a, b0, lane, first);
    return chunks == 0 ? 0 : splits_of(a, cps, chunks).used;
  };
  int total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) total += wave_total(splits(b0));
  const int head = id / total;
  if (head >= a.Hkv) return {-1, 0};
  const int at = id - head * total;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = splits(b0), incl = wave_prefix(n);
    const unsigned long long in = __ballot(at < before + incl);
    if (in != 0) {
      const int l = __ffsll(in) - 1;
      return {(b0 + l) * a.Hkv + a.Hkv - 1 - head, at - before - (__shfl(incl, l, 64) - __shfl(n, l, 64))};
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return {-1, 0};
}

template <typename T, typename F, int D>
__global__ __launch_bounds__(kTree8Threads, (Tree8Cfg<T, D>::WGS_PER_CU)) void coalibi_tree8_kernel(Tree8Args a8) {
  using C = Tree8Cfg<T, D>;
  using M = Mfma<T>;
  using V8 = typename M::vec8;
  constexpr int DT = C::DT;
  constexpr bool kCodesTakeScales = __is_same(T, _Float16);
  constexpr int kMostPower = __is_same(F, E4M3) ? 7 : 5, kLeastPower = __is_same(F, E4M3) ? -15 : -20;  // (TimesPower)
  const TreeArgs& a = a8.t;
  __shared__ __align__(16) char smem[C::LDS_BYTES];
  __shared__ float sMax[kTree8Waves][32], sSum[kTree8Waves][32], sSig[kTree8Waves][32], sScale[kTree8Waves][32];
  __shared__ bool sLost[kTree8Waves];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane & 31, hh = lane >> 5;
  // Ids: the row blocks of an item (split, sequence, kv head) 8 apart, so that they share an XCD and its L2.
  const int RB = a.row_blocks, id = blockIdx.x;
  const int rb = (id >> 3) % RB, item = (id / (8 * RB)) * 8 + (id & 7);
  const int nS = a.nSplits;
  int cps = a.cps;
  TreeItem it;
  if (a.plan) {
    const int first = lane_chunks(a, lane);
    cps = plan_cps(a, lane, first);
    it = head_item(a, cps, item, lane, first);
  } else {
    const int per_head = a.B * nS, head = item / per_head, at = item - head * per_head;
    it = head < a.Hkv ? TreeItem{at / nS * a.Hkv + a.Hkv - 1 - head, at % nS} : TreeItem{-1, 0};
  }
  const int bhk = __builtin_amdgcn_readfirstlane(it.bhk), split = __builtin_amdgcn_readfirstlane(it.split);
  if (bhk < 0) return;
  const int b = __builtin_amdgcn_readfirstlane(bhk / a.Hkv), hkv = bhk - b * a.Hkv;
  const int L = __builtin_amdgcn_readfirstlane(filled_rows(a, b));
  const int chunks = __builtin_amdgcn_readfirstlane(chunks_of(a, L));
  TreeSplits sp = splits_of(a, cps, chunks);
  sp = {__builtin_amdgcn_readfirstlane(sp.cps), __builtin_amdgcn_readfirstlane(sp.used)};
  if (split >= sp.used) return;
  const bool newest = split == sp.used - 1;

  // The split's tiles: of the filled rows, then (in the newest) of the new keys, shared out over the wavefronts in order.
  const int cache_tiles = (L + 31) >> 5, fresh_tiles = (a.T + 31) >> 5, per_chunk = a.chunk >> 5;
  const int t0 = min(split * sp.cps * per_chunk, cache_tiles);
  const int t1 = newest ? cache_tiles + fresh_tiles : min((split + 1) * sp.cps * per_chunk, cache_tiles);
  const int per = (t1 - t0 + kTree8Waves - 1) / kTree8Waves;
  const int t_first = min(t0 + wave * per, t1), t_end = min(t_first + per, t1);

  const int R = a.G * a.T, row = rb * 32 + hl;
  const bool row_ok = row < R;
  const int rsafe = row_ok ? row : 0;
  const int g = rsafe / a.T, t = rsafe - g * a.T, h = hkv * a.G + g;
  const float lam2 = a.slopes[h] * kLog2e;

  unsigned long long sees = 0;
  if (newest) {
    if (tid == 0 && nS > 1) a.used[bhk] = sp.used;  // every row block writes the same
    const unsigned long long all = ancestors(a, b, lane);
    sees = (unsigned long long)__shfl((unsigned)(all >> 32), t, 64) << 32 | __shfl((unsigned)all, t, 64);
  }

  const T* const kn = head_at(static_cast<const T*>(a.k), a.kl, b, hkv);
  const T* const vn = head_at(static_cast<const T*>(a.v), a.vl, b, hkv);
  const char* const kc = static_cast<const char*>(a.kc) + (size_t)hkv * a.kcl.h;
  const char* const vc = static_cast<const char*>(a.vc) + (size_t)hkv * a.vcl.h;
  const float* const ksc = a8.ks + (size_t)hkv * a8.ksh;
  const float* const vsc = a8.vs + (size_t)hkv * a8.vsh;
  const int page_mask = a.place.table != nullptr ? (1 << a.place.page_shift) - 1 : 0x7fffffff;

  // The table entries of a tile's two blocks of 16 rows (of the last filled row past it).  They are looked at when they are used:
  // an entry outside the pool is read as unit 0, and makes the sequence NaN.
  struct Units {
    int u[2];
  };
  const int* const table = a.place.table + (size_t)b * a.place.table_stride;
  auto find = [&](int tile) {
    Units f{{b, b}};
    if (a.place.table != nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i) f.u[i] = scalar_load(table + (min(tile * 32 + 16 * i, L - 1) >> a.place.page_shift));
    }
    return f;
  };
  bool lost = false;
  auto check = [&](Units& f) {
    if (a.place.table != nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = (unsigned)f.u[i] < (unsigned)a.place.units;
        lost |= !in;
        f.u[i] = in ? f.u[i] : 0;
      }
    }
  };
  // A cached tile's loads.  CLAMP: rows past the filled ones are read from the last of them (their scores are masked).  Every lane
  // reads from one of the tile's two blocks: their addresses are the wavefront's, and a lane picks.
  const int krow = kRowOfReg(hl);
  auto pick = [](bool second, const auto* p0, const auto* p1) {
    const auto a0 = (unsigned long long)p0, a1 = (unsigned long long)p1;
    const unsigned lo = second ? (unsigned)a1 : (unsigned)a0, hi = second ? (unsigned)(a1 >> 32) : (unsigned)(a0 >> 32);
    return (decltype(p0))((unsigned long long)hi << 32 | lo);
  };
  auto load_keys = [&](auto clamp, int tile, const Units& f, Keys8<D>& x) {
    const int key0 = tile * 32;
    const int key = decltype(clamp)::value ? min(key0 + krow, L - 1) : key0 + krow;
    const char* const p = pick(krow >= 16, kc + (size_t)f.u[0] * a.kcl.b, kc + (size_t)f.u[1] * a.kcl.b) +
                          (size_t)(key & page_mask) * D + hh * (D < 32 ? 8 : 16);
    if constexpr (D < 32) {
      const u32x2 lo = *reinterpret_cast<const u32x2*>(p);
      x.k[0] = u32x4{lo[0], lo[1], 0, 0};
    } else {
#pragma unroll
      for (int i = 0; i < Keys8<D>::KL; ++i) x.k[i] = ld16(p + 32 * i);
    }
    const int r1 = decltype(clamp)::value ? min(key0 + 16, L - 1) : key0 + 16;
    const int at0 = (key0 & page_mask) >> 4, at1 = (r1 & page_mask) >> 4;
    x.ks = *pick(hh != 0, ksc + (size_t)f.u[0] * a8.ksb + at0, ksc + (size_t)f.u[1] * a8.ksb + at1);
    x.vs = *pick(hh != 0, vsc + (size_t)f.u[0] * a8.vsb + at0, vsc + (size_t)f.u[1] * a8.vsb + at1);
  };
  auto load_values = [&](auto clamp, int tile, const Units& f, Run<DT> (&v)[16]) {
    const int r0 = tile * 32, r1 = decltype(clamp)::value ? min(r0 + 16, L - 1) : r0 + 16;
    const char* const p = pick(hh != 0, vc + (size_t)f.u[0] * a.vcl.b + (size_t)(r0 & page_mask) * D,
                               vc + (size_t)f.u[1] * a.vcl.b + (size_t)(r1 & page_mask) * D) +
                          (D < 32 ? hl & 15 : DT * hl);
    const int left = L - 1 - (hh ? r1 : r0);  // (clamped)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i].load(p + (decltype(clamp)::value ? min(i, left) : i) * D);
  };
  using Inside = std::false_type;
  using Clamped = std::true_type;

  // Q^T fragments in the order of K's: step 2 i + s holds the elements 32 i + 16 (l / 32) + 8 s + e of the row (D 16: 8 (l / 32)
  // + e).  Past R they are the first row's, and come to nothing.
  V8 qf[C::KS];
  {
    const T* const q = head_at(static_cast<const T*>(a.q), a.ql, b, h) + (size_t)t * a.ql.r;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks)
      qf[ks] = ld_vec8(q + (D < 32 ? 8 * hh : (ks >> 1) * 32 + 16 * hh + (ks & 1) * 8));
  }

  // State of the lane's row: scale, this half's share of the sum, O^T, and the sigma of the keys after the current ones.
  float m2 = kNegInf, lsum = 0.f, carry = 0.f;
  // Weights of the last tile, rounded to q's type for their product with V (their sum is not), as the other attentions of this library
  // round them.  In two parts, the second what the first leaves, o has no rounding but its own, and it costs 6 % of the drafts and of
  // the single token, 4 % of the 32 sequences.
  V8 pb[2];
  f32x16 acc[DT];  // in units of 2^unit
  int unit = 0, power = 0;  // power: of the lane's codes of the tile whose values are held
  bool first_scale = true;
#pragma unroll
  for (int j = 0; j < DT; ++j) acc[j] = f32x16{};

  // From a tile's scores (log2 units; -inf where the row does not see the key) to its weights, in the order of P^T; without `near`
  // only its sigmas count.
  auto weigh_or_pass = [&](f32x16 s, float vs, bool near) {
    float loc[16], run = 0.f;
#pragma unroll
    for (int r = 15; r >= 0; --r) {
      run += sigmoid_log2(s[r]);
      loc[r] = run;
    }
    const float oth = other_half(run), before = carry;
    carry += hh ? run + oth : oth + run;
    if (!near) return;
    const float mb = m2 == kNegInf ? 0.f : m2;
    const float cst = mb + lam2 * (before + (hh ? 0.f : oth)) - __builtin_amdgcn_logf(vs);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(-lam2, loc[r], s[r] - cst);
    auto weights = [&] {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x8 p;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = fast_exp2(s[8 * i + e]);
          sum += p[e];  // before the rounding for the product: the LSE is fp32's
        }
        pb[i] = M::pack(p);
      }
      return sum;
    };
    float sum = weights();
    if (__any(m2 == kNegInf || sum > kTreeRescale)) {
      float mt = kNegInf;
#pragma unroll
      for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[r]);
      mt = fmaxf(mt, other_half(mt));
      const bool need = mt > (m2 == kNegInf ? kNegInf : 0.f);
      const float delta = need ? mt : 0.f;
      const float alpha = need ? (m2 == kNegInf ? 0.f : fast_exp2(-delta)) : 1.f;
      m2 = need ? mb + delta : m2;
      lsum *= alpha;
#pragma unroll
      for (int j = 0; j < DT; ++j) acc[j] *= alpha;
      s -= delta;
      sum = weights();
    }
    lsum = fmaf(sum, fast_rcp(vs), lsum);
  };
  auto weigh = [&](f32x16 s, float vs) { weigh_or_pass(s, vs, true); };

  // The scores of a tile of cached keys, in log2 units.
  auto scores = [&](const Keys8<D>& x) {
    f32x16 s{};
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      const unsigned lo = x.k[ks >> 1][2 * (ks & 1)], hi = x.k[ks >> 1][2 * (ks & 1) + 1];
      s = M::k16(code_vec8<T, F>(lo, hi), qf[ks], s);
    }
    const float sc = a.sc2 * x.ks;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= sc;
    return s;
  };
  auto scale_of = [&](const Keys8<D>& x) {
    const bool fine = scale_ok(x.ks) && scale_ok(x.vs);
    lost |= !fine;
    return fine ? x.vs : 1.f;
  };
  // What the weights take of a tile's scales of V.  fp16's have little room below the row's largest (subnormal below 2^-14), so there the
  // codes take the scales' powers of two, relative to a unit of O that rises with the largest, as far as their products are exact
  // (2^22 below it for e4m3, 2^25 for int8); the weights what is left, from 1 to 2.
  auto take = [&](float vs) {
    if constexpr (!kCodesTakeScales) return vs;
    const int e = (int)(__builtin_bit_cast(unsigned, vs) >> 23) - 127;
    const int most = max(__builtin_amdgcn_readlane(e, 0), __builtin_amdgcn_readlane(e, 32));
    if (first_scale || most - unit > kMostPower) {
      const int to = most - kMostPower;
      const float f = ldexpf(1.f, unit - to);
#pragma unroll
      for (int j = 0; j < DT; ++j) acc[j] *= f;
      unit = to;
      first_scale = false;
    }
    power = max(e - unit, kLeastPower);
    return ldexpf(vs, -(unit + power));
  };
  auto add_values = [&](const Run<DT> (&v)[16], const V8 (&pb)[2]) {
    using By = std::conditional_t<kCodesTakeScales, TimesPower<F>, Times1>;
    const By by(power);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int q4 = 0; q4 < (DT + 3) / 4; ++q4) {
        unsigned w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = v[8 * st + e].w[q4];
        acc[4 * q4] = M::k16(byte_vec8<T, F, 0>(w, by), pb[st], acc[4 * q4]);
        if constexpr (DT > 1) acc[4 * q4 + 1] = M::k16(byte_vec8<T, F, 1>(w, by), pb[st], acc[4 * q4 + 1]);
        if constexpr (DT > 2) {
          acc[4 * q4 + 2] = M::k16(byte_vec8<T, F, 2>(w, by), pb[st], acc[4 * q4 + 2]);
          acc[4 * q4 + 3] = M::k16(byte_vec8<T, F, 3>(w, by), pb[st], acc[4 * q4 + 3]);
        }
      }
    }
  };

  int tile = t_end - 1;
  const int whole = min(t_end, L >> 5) - 1;  // the newest tile of filled rows alone
  Keys8<D> ka, kb;
  Run<DT> v[16];
  Units ua{}, ub{};
  if (whole >= t_first) {
    ua = find(whole);
    check(ua);
    load_keys(Inside{}, whole, ua, ka);
    ub = find(max(whole - 1, t_first));
  }
  // The new keys' tiles.
  for (; tile >= t_first && tile >= cache_tiles; --tile) {
    const int key0 = (tile - cache_tiles) * 32;
    f32x16 s{};
    {
      const T* const k = kn + (size_t)min(key0 + krow, a.T - 1) * a.kl.r;
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks)
        s = M::k16(ld_vec8(k + (D < 32 ? 8 * hh : (ks >> 1) * 32 + 16 * hh + (ks & 1) * 8)), qf[ks], s);
    }
    const unsigned ok = (unsigned)(sees >> (key0 + 16 * hh));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = ok >> r & 1 ? s[r] * a.sc2 : kNegInf;
    weigh(s, 1.0f);
    // A product with a weight of 0 would carry an infinity or a NaN of a value to rows that do not see it: such values are 0
    // here and added to the rows that do below.
    unsigned bad = 0;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      typedef T row_t __attribute__((ext_vector_type(DT)));
      row_t x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = *reinterpret_cast<const row_t*>(vn + (size_t)min(key0 + 16 * hh + 8 * st + e, a.T - 1) * a.vl.r +
                                               (D < 32 ? hl & 15 : DT * hl));
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        V8 va;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          T y = x[e][j];
          if (not_finite(y)) {
            y = T(0);
            bad |= 1u << (16 * hh + 8 * st + e);
          }
          va[e] = y;
        }
        acc[j] = M::k16(va, pb[st], acc[j]);
      }
    }
    if (__any(bad != 0)) {
      for (int key = 0; key < min(a.T - key0, 32); ++key) {
        if (!__any(bad >> key & 1)) continue;
        if (sees >> (key0 + key) & 1) {
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = DT * ((r >> 2) * 8 + hh * 4 + (r & 3)) + j;
              if (d >= D) continue;
              const T x = vn[(size_t)(key0 + key) * a.vl.r + d];
              if (not_finite(x)) acc[j][r] += static_cast<float>(x);
            }
        }
      }
    }
  }
  // The tile that the filled rows end in.
  if (tile > whole && tile >= t_first) {
    Units f = find(tile);
    check(f);
    load_keys(Clamped{}, tile, f, kb);
    load_values(Clamped{}, tile, f, v);
    f32x16 s = scores(kb);
    const int left = L - tile * 32 - 16 * hh;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = r < left ? s[r] : kNegInf;
    weigh(s, take(scale_of(kb)));
    add_values(v, pb);
    --tile;
  }
  // The others.  Keys come in a tile ahead and table entries two; a tile's values while it is weighed and the next one's scores
  // are taken, which is when its own product with the weights follows.
  bool held = false;  // such a product is due
  auto step = [&](Keys8<D>& x, Keys8<D>& next) {
    const Units f = ua;
    if (tile > t_first) {
      ua = ub;
      check(ua);
      load_keys(Inside{}, tile - 1, ua, next);
      ub = find(max(tile - 2, t_first));
    }
    f32x16 s = scores(x);
    if (held) add_values(v, pb);
    // A tile whose keys all weigh less than 2^-a.far of their row's sum, as far as it is known, is left out but for its sigmas: a_j
    // is at most its score less the sigmas after the tile.  A NaN keeps it: the largest score is NaN if one is (v_maximum3; fmaxf
    // takes the other operand).
    float mt = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = __builtin_elementwise_maximum(mt, s[r]);
    held = __any(row_ok && !(lam2 >= 0.f && mt - lam2 * carry - m2 < __builtin_amdgcn_logf(lsum) - a.far));
    if (held) load_values(Inside{}, tile, f, v);
    float vs = scale_of(x);
    if (held) vs = take(vs);
    weigh_or_pass(s, vs, held);
    --tile;
  };
  while (tile >= t_first) {
    step(ka, kb);
    if (tile < t_first) break;
    step(kb, ka);
  }
  if (held) add_values(v, pb);

  // The wavefronts joined: each one's maximum shifted by the sigmas of the later ones' keys.
  const float l = lsum + other_half(lsum);
  const bool any_lost = __any(lost);
  if (lane == 0) sLost[wave] = any_lost;
  if (hh == 0) {
    sMax[wave][hl] = m2;
    sSum[wave][hl] = l;
    sSig[wave][hl] = carry;
  }
  __syncthreads();
  if (tid < 32) {  // lane tid holds row tid
    float after = 0.f, m = kNegInf, mw[kTree8Waves];
    bool gone = false;
#pragma unroll
    for (int w = kTree8Waves - 1; w >= 0; --w) {
      mw[w] = sMax[w][tid] - lam2 * after;
      after += sSig[w][tid];
      m = fmaxf(m, mw[w]);
      gone |= sLost[w];
    }
    float ls = 0.f, f[kTree8Waves];
#pragma unroll
    for (int w = 0; w < kTree8Waves; ++w) {
      const bool none = mw[w] == kNegInf;
      f[w] = none ? 0.f : fast_exp2(mw[w] - m);
      ls += none && sSum[w][tid] == 0.f ? 0.f : f[w] * sSum[w][tid];
    }
    // The sum to [1, 2): the merge takes it for at least 1, and the scales of V have moved it.
    const int e = ls > 0.f && ls < __builtin_inff() ? __builtin_amdgcn_frexp_expf(ls) - 1 : 0;
#pragma unroll
    for (int w = 0; w < kTree8Waves; ++w) sScale[w][tid] = ldexpf(f[w], -e);
    sMax[0][tid] = m + static_cast<float>(e);
    sSum[0][tid] = gone ? __builtin_nanf("") : ldexpf(ls, -e);
    sSig[0][tid] = after;
  }
  __syncthreads();
  float* const so = reinterpret_cast<float*>(smem) + (size_t)wave * 32 * C::LDO + hl * C::LDO;
  const float f = ldexpf(sScale[wave][hl], unit);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int d = DT * ((r >> 2) * 8 + hh * 4 + (r & 3));
    if (d < D) {
#pragma unroll
      for (int j = 0; j < DT; ++j) so[d + j] = acc[j][r] * f;
    }
  }
  const size_t row0 = (size_t)bhk * R + rb * 32;  // the block's first row in o, lse and the partials
  const int rows = min(R - rb * 32, 32);
  const bool direct = sp.used == 1;
  if (wave == 0 && hh == 0 && row_ok) {
    const bool absent = newest && sees == 0;
    if (direct) {
      const float ls = sSum[0][hl];
      if (a.lse != nullptr) a.lse[row0 + hl] = absent ? kNegInf : (sMax[0][hl] + log2f(ls)) * kLn2;
      sSig[1][hl] = absent ? 0.f : 1.f / ls;
      sMax[1][hl] = absent ? 0.f : 1.f;
    } else {
      const size_t pi = (row0 + hl) * nS + split;
      a.pmax[pi] = sMax[0][hl];
      a.psum[pi] = absent ? kAbsent : sSum[0][hl];
      a.psig[pi] = sSig[0][hl];
    }
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += kTree8Threads) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    f32x4 s = f32x4{};
#pragma unroll
    for (int w = 0; w < kTree8Waves; ++w)
      s += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(smem) + ((size_t)w * 32 + r) * C::LDO + d);
    if (direct) {
      typedef T out4 __attribute__((ext_vector_type(4)));
      const bool there = sMax[1][r] != 0.f;
      const float inv = sSig[1][r];
      out4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(there ? s[e] * inv : 0.f);
      *reinterpret_cast<out4*>(static_cast<T*>(a.o) + (row0 + r) * D + d) = v;
    } else {
      *reinterpret_cast<f32x4*>(a.pout + ((row0 + r) * nS + split) * D + d) = s;
    }
  }
}

}  // namespace

template <typename T, typename F, int D>
hipError_t launch_tree8(const Tree8Args& a8, hipStream_t stream) {
  const TreeArgs& a = a8.t;
  // Under a plan at most one round of work-groups and a rounded-up split per sequence.
  const long long even = (long long)a.B * a.Hkv * a.nSplits;
  const long long items = a.plan ? std::min<long long>(even, ((long long)a.share + a.B) * a.Hkv) : even;
  const dim3 grid(static_cast<unsigned>((items + 7) / 8 * 8 * a.row_blocks));
  hipLaunchKernelGGL((coalibi_tree8_kernel<T, F, D>), grid, dim3(kTree8Threads), 0, stream, a8);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || a.nSplits == 1 ? e : launch_tree_merge<T, D>(a, stream);
}

#define COALIBI_INST_TREE8(T, D)                                                 \
  template hipError_t launch_tree8<T, E4M3, D>(const Tree8Args&, hipStream_t);   \
  template hipError_t launch_tree8<T, I8, D>(const Tree8Args&, hipStream_t);
COALIBI_INST_TREE8(_Float16, 16)
COALIBI_INST_TREE8(_Float16, 32)
COALIBI_INST_TREE8(_Float16, 64)
COALIBI_INST_TREE8(_Float16, 128)
COALIBI_INST_TREE8(_Float16, 256)
COALIBI_INST_TREE8(__bf16, 16)
COALIBI_INST_TREE8(__bf16, 32)
COALIBI_INST_TREE8(__bf16, 64)
COALIBI_INST_TREE8(__bf16, 128)
COALIBI_INST_TREE8(__bf16, 256)
COALIBI_INST_TREE8(float, 16)
COALIBI_INST_TREE8(float, 32)
COALIBI_INST_TREE8(float, 64)
COALIBI_INST_TREE8(float, 128)

}  // namespace coalibi
