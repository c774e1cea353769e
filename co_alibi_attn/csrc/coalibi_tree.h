// Device code that the tree decodes share: over caches of the input type (coalibi_tree.hip) and of 8 bits (coalibi_tree8.hip).
#pragma once
#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

// O is rescaled when the weights of a lane's keys of a chunk sum to more than this at the running scale: a weight stays
// far below fp16's 65504.  (A maximum per chunk in its place: 77 us against 75, 96 rows over 16 sequences of 8192 keys.)
constexpr float kTreeRescale = 4096.0f;

// A partial's sum in the newest split where the row's node is absent.
constexpr float kAbsent = -1.0f;

// Inclusive sum over the lanes up to each one, by DPP moves (shuffles take an LDS round trip a step).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_prefix(int x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4 and 8 within 16 lanes
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // the 16 lanes before
  return dpp_add<0x143, 0xc>(x);  // the 32 lanes before
}
// The largest of the lanes' values (>= 0), in the same steps.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_largest(int x) {
  x = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(x))));
  return __builtin_amdgcn_readlane(dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(x)), 63);
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_prefix(x), 63); }

__device__ __forceinline__ int filled_rows(const TreeArgs& a, int b) {
  return a.seq_lens == nullptr ? a.L : min(max(a.seq_lens[b], 0), a.L);
}
// A sequence's chunks: of its filled rows, and the new keys' (the last).
__device__ __forceinline__ int chunks_of(const TreeArgs& a, int len) { return (len + a.chunk - 1) / a.chunk + 1; }

// The chunks of sequence b0 + lane; `first`: those of the first 64, which the plan's loops read once.  (The loads and divisions of a
// plan made anew at each trial: 83.8 us against 81.5, 96 rows over 16 sequences.)
__device__ __forceinline__ int lane_chunks(const TreeArgs& a, int b) { return b < a.B ? chunks_of(a, filled_rows(a, b)) : 0; }
__device__ __forceinline__ int lane_chunks(const TreeArgs& a, int b0, int lane, int first) {
  return b0 == 0 ? first : lane_chunks(a, b0 + lane);
}

// The sequences' splits together, of cps chunks each.
__device__ __forceinline__ int total_splits(const TreeArgs& a, int cps, int lane, int first) {
  int n = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) n += wave_total((unsigned)(lane_chunks(a, b0, lane, first) + cps - 1) / (unsigned)cps);
  return n;
}

// Chunks per split of a launch with a plan (every wavefront computes the same): the splits share out the batch's real
// chunks over one round of `share` work-groups per kv head and row block.  An equal share of the chunks each, or up
// to 3/8 more and one where the rounded-up splits then fit the round.
__device__ __forceinline__ int plan_cps(const TreeArgs& a, int lane, int first) {
  int total = 0, longest = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = lane_chunks(a, b0, lane, first);
    total += wave_total(n);
    longest = max(longest, wave_largest(n));
  }
  // No more than nSplits of any sequence.
  const int c0 = max((total + a.share - 1) / a.share, (longest + a.nSplits - 1) / a.nSplits);
  for (int c = c0; c <= c0 + 1 + c0 * 3 / 8; c += 1 + c / 16)
    if (total_splits(a, c, lane, first) <= a.share) return c;
  return c0;
}

// A sequence's splits: `used` of them, of cps chunks each (the last may have fewer).
struct TreeSplits {
  int cps, used;
};
__device__ __forceinline__ TreeSplits splits_of(const TreeArgs& a, int cps, int chunks) {
  if (a.plan) {  // as many as the plan's cps make, then of equal length
    const unsigned n = (unsigned)(chunks + cps - 1) / (unsigned)cps;
    cps = (int)((chunks + n - 1) / n);
  }
  return {cps, (int)((unsigned)(chunks + cps - 1) / (unsigned)cps)};
}

// The (sequence and kv head, split) of item `id` under a plan: items run over the sequences' own splits, split
// fastest; ids past the last one have none (bhk < 0).
struct TreeItem {
  int bhk, split;
};
__device__ __forceinline__ TreeItem plan_item(const TreeArgs& a, int cps, int id, int lane, int first) {
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int chunks = lane_chunks(a, b0, lane, first), n = chunks == 0 ? 0 : splits_of(a, cps, chunks).used;
    const int incl = wave_prefix(n * a.Hkv);
    const unsigned long long in = __ballot(id < before + incl);
    if (in != 0) {
      const int l = __ffsll(in) - 1;
      const int splits = __shfl(n, l, 64), at = id - before - (__shfl(incl, l, 64) - splits * a.Hkv);
      const int hkv = at / splits;
      return {__builtin_amdgcn_readfirstlane((b0 + l) * a.Hkv + hkv), __builtin_amdgcn_readfirstlane(at - hkv * splits)};
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return {-1, 0};
}

// Lane t: the new keys that node t sees (bit j: key j), or 0 for an absent node -- one whose chain of parents
// leaves [-1, own index).  Six steps of doubling: after step i a lane has gathered 2^i ancestors.
__device__ __forceinline__ unsigned long long ancestors(const TreeArgs& a, int b, int lane) {
  if (a.parents == nullptr) return lane == 63 ? ~0ull : (2ull << lane) - 1;
  const int p = lane < a.T ? a.parents[(size_t)b * a.parents_stride + lane] : -1;
  const bool valid = p >= -1 && p < lane;
  unsigned lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
  int bad = valid ? 0 : 1, up = valid ? p : -1;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int from = max(up, 0);
    const unsigned olo = __shfl(lo, from, 64), ohi = __shfl(hi, from, 64);
    const int obad = __shfl(bad, from, 64), oup = __shfl(up, from, 64);
    if (up >= 0) {
      lo |= olo;
      hi |= ohi;
      bad |= obad;
      up = oup;
    }
  }
  return bad ? 0ull : (unsigned long long)hi << 32 | lo;
}

// A wave-uniform int from the constant address space: a scalar load, whatever the memory clobbers around it.
__device__ __forceinline__ int scalar_load(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(size_t)p;
}

template <typename T>
__device__ __forceinline__ bool not_finite(T x) {
  if constexpr (sizeof(T) == 4) return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u;
  constexpr unsigned exp_bits = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  if constexpr (sizeof(T) == 2) return (__builtin_bit_cast(unsigned short, x) & exp_bits) == exp_bits;
}

}  // namespace

}  // namespace coalibi
