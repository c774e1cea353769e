// Co-ALiBi attention of a step's new tokens -- one token, a run of them or a tree of drafts -- over a key /
// value cache and each other, on gfx950.
//
// Node t of a sequence sees the cache's filled rows and, after them, its chain of ancestors up to itself.
// Parents come before their children, so those of the T new keys that a node sees stand in index order
// and are the bits of a 64-bit mask.  With the keys in this order, as in the decode (coalibi_decode.hip):
//   t_j = sm_scale*log2(e) * q.k_j,   sigma_j = sigmoid(t_j / log2(e)),
//   z_j = sum_{k >= j} sigma_k,       a_j = t_j - slope*log2(e) * z_j,
//   O   = sum_j 2^(a_j - m) v_j / sum_j 2^(a_j - m),   LSE = (m + log2 l) * ln 2.
//
// The R = G*T query rows of a kv head (row g*T + t) read the same keys, so a work-group takes up to 128 of them
// over a run of key chunks (a split), from its newest chunk to its oldest; the sequence's newest chunk is
// the new keys, masked by the ancestor bits.  Splits know only their own keys' z; the merge shifts each
// one's maximum by the sigma of the splits after it (as the decode's does).
// The four wavefronts of a work-group are laid out by R: WR of them over 32-row tiles and 4 / WR over the
// chunk's keys, so that small R still has four wavefronts of key tiles and large R reads each tile once for 128 rows.
//   S^T = K Q^T and O^T += V^T P^T on MFMA, keys on the accumulator rows of S^T (in the kRowOfReg order: a lane holds 16
// consecutive keys of one query row, so the suffix sums are register-local) and query rows on the
// columns of both, so every per-row factor is a lane's own.  K and V come in by buffer-to-LDS DMA, one chunk ahead.
// Where wavefronts share the tiles of all keys (WR 4) there are two buffers of 64 keys and one barrier per chunk; else
// one buffer of 128 keys, each tile's next chunk issued as soon as the tile has been read.  LDS rows are not
// padded: the 16-byte pieces of a row are stored in an order XORed with its index (the DMA lanes fetch them so), which
// keeps the operand reads off each other's banks and every DMA lane busy.
//
// What bounds it, bf16 or fp16 at D 128, captured: 64 query rows over 8192 keys 19.5 us, latency (the merge 4 of it,
// three chunks in a row the rest; VALU issues in 11 % of the cycles, MFMA in 4 %); 96 rows over 16 sequences of up to 8192
// keys 75 us, of which the split 68 (265 MB fetched at 3.9 TB/s, VALU 35 %, MFMA 13 %; 259 MB are 38 us at the read rate of 6.9
// TB/s); 256 rows over 131072 keys 191 to 197 us from box to box (VALU 46 %, MFMA 20 %, 3.0 TB/s; 538 MB are 78 us, 137 Gflop
// of products 113).
//   In the 128-row form nothing is saturated: a wavefront's products, two exponentials, a reciprocal and suffix sums per
// score follow one another behind one barrier per 64 keys, and the two wavefronts of a SIMD run in step.  Leaving out the
// chunks of far keys took 217 us to 187.
//   Smaller blocks wait rather than issue, and looking for far chunks made them slower (19.7 -> 20.3 us at 64 rows).
#include <algorithm>
#include <type_traits>

#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
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

// The sequences' splits together, of cps chunks each.
__device__ __forceinline__ int total_splits(const TreeArgs& a, int cps, int lane) {
  int n = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64)
    n += wave_total(b0 + lane < a.B ? (chunks_of(a, filled_rows(a, b0 + lane)) + cps - 1) / cps : 0);
  return n;
}

// Chunks per split of a launch with a plan (every wavefront computes the same): the splits share out the batch's real
// chunks over one round of `share` work-groups per kv head and row block.  An equal share of the chunks each, or up
// to 3/8 more and one where the rounded-up splits then fit the round.
__device__ __forceinline__ int plan_cps(const TreeArgs& a, int lane) {
  int total = 0, longest = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? chunks_of(a, filled_rows(a, b0 + lane)) : 0;
    total += wave_total(n);
    longest = max(longest, wave_largest(n));
  }
  // No more than nSplits of any sequence.
  const int c0 = max((total + a.share - 1) / a.share, (longest + a.nSplits - 1) / a.nSplits);
  for (int c = c0; c <= c0 + 1 + c0 * 3 / 8; c += 1 + c / 16)
    if (total_splits(a, c, lane) <= a.share) return c;
  return c0;
}

// A sequence's splits: `used` of them, of cps chunks each (the last may have fewer).
struct TreeSplits {
  int cps, used;
};
__device__ __forceinline__ TreeSplits splits_of(const TreeArgs& a, int cps, int chunks) {
  if (a.plan) {  // as many as the plan's cps make, then of equal length
    const int n = (chunks + cps - 1) / cps;
    cps = (chunks + n - 1) / n;
  }
  return {cps, (chunks + cps - 1) / cps};
}

// The (sequence and kv head, split) of item `id` under a plan: items run over the sequences' own splits, split
// fastest; ids past the last one have none (bhk < 0).
struct TreeItem {
  int bhk, split;
};
__device__ __forceinline__ TreeItem plan_item(const TreeArgs& a, int cps, int id, int lane) {
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < a.B ? splits_of(a, cps, chunks_of(a, filled_rows(a, b))).used : 0;
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

template <typename T, int D>
struct TreeCfg {
  static constexpr int E = sizeof(T);
  static constexpr int ROWB = D * E;       // bytes per key in LDS
  static constexpr int CPR = ROWB / 16;    // 16-byte pieces of them
  static constexpr int KS = D / 16;        // k16 steps over the head dim
  static constexpr int DT = D < 32 ? 1 : D / 32;  // 32-row tiles of O^T
  static constexpr int HALF_INSTR = 16 * ROWB >= 1024 ? 16 * ROWB / 1024 : 1;  // DMA instructions per 16 keys
  static constexpr int TILES = 2 * kTreeLdsKeys * ROWB;  // bytes of the K and V buffers
  // At the end the wavefronts' O rows (fp32, rows 16 bytes apart from a power of two) alias the chunks.
  static constexpr int LDO = D + 4;
  static constexpr int O_BYTES = kTreeWaves * 32 * LDO * 4;
  static constexpr int LDS_BYTES = TILES > O_BYTES ? TILES : O_BYTES;
  static constexpr int WGS_PER_CU = LDS_BYTES <= 76 * 1024 ? 2 : 1;
};

// The XOR of a key's piece order, by the key's index in its 32-key tile.  K: a read pass is 16 bytes of 16
// consecutive A-operand rows R (key kRowOfReg(R)).  V: a transpose read's pass is 64 bytes of 4 consecutive
// keys; fp32 reads 128 bytes of keys k and k + 16.  A pass covers the 64 banks (256 bytes) once.
template <int CPR>
__device__ __forceinline__ constexpr int swizzle_k(int R) {
  return CPR >= 16 ? R & 15 : CPR == 8 ? (R >> 1) & 7 : CPR == 4 ? (R >> 2) & 3 : (R >> 3) & 1;
}
template <int CPR, int E>
__device__ __forceinline__ constexpr int swizzle_v(int key) {
  if (E == 4) return CPR >= 16 ? ((key >> 4) & 1) << 3 : 0;
  return CPR >= 16 ? (key & 3) << 2 : CPR == 8 ? ((key >> 1) & 1) << 2 : 0;
}

// N buffer-to-LDS DMA instructions at LDS byte address lds, lds + 1024, ..., ordered by the caller's waits
// (dma16_to_lds_untracked's rules); one run, so that only the first waits out the writes of its scalar operands.
// Every m0 comes from the scalar address: added to itself, m0 lost its upper bits for LDS addresses past 64 KB.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
#define COALIBI_DMA_FIRST(V, NT) "s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 " V ", %1, 0 offen" NT " lds"
#define COALIBI_DMA_NEXT(V, AT, NT) "\n\ts_add_u32 m0, %0, " AT "\n\ts_nop 0\n\tbuffer_load_dwordx4 " V ", %1, 0 offen" NT " lds"
#define COALIBI_DMA1(NT) COALIBI_DMA_FIRST("%2", NT)
#define COALIBI_DMA2(NT) COALIBI_DMA1(NT) COALIBI_DMA_NEXT("%3", "0x400", NT)
#define COALIBI_DMA4(NT) COALIBI_DMA2(NT) COALIBI_DMA_NEXT("%4", "0x800", NT) COALIBI_DMA_NEXT("%5", "0xc00", NT)
template <int N, bool NT>
__device__ __forceinline__ void dma_run(__amdgpu_buffer_rsrc_t r, unsigned lds, const int* v) {
  if constexpr (N == 1 && NT) {
    asm volatile(COALIBI_DMA1(" nt")::"s"(lds), "s"(r), "v"(v[0]) : "memory", "m0");
  } else if constexpr (N == 1) {
    asm volatile(COALIBI_DMA1("")::"s"(lds), "s"(r), "v"(v[0]) : "memory", "m0");
  } else if constexpr (N == 2 && NT) {
    asm volatile(COALIBI_DMA2(" nt")::"s"(lds), "s"(r), "v"(v[0]), "v"(v[1]) : "memory", "m0", "scc");
  } else if constexpr (N == 2) {
    asm volatile(COALIBI_DMA2("")::"s"(lds), "s"(r), "v"(v[0]), "v"(v[1]) : "memory", "m0", "scc");
  } else if constexpr (N == 4 && NT) {
    asm volatile(COALIBI_DMA4(" nt")::"s"(lds), "s"(r), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]) : "memory", "m0", "scc");
  } else if constexpr (N == 4) {
    asm volatile(COALIBI_DMA4("")::"s"(lds), "s"(r), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]) : "memory", "m0", "scc");
  } else {
    dma_run<N / 2, NT>(r, lds, v);
    dma_run<N / 2, NT>(r, lds + N / 2 * 1024, v + N / 2);
  }
}
#undef COALIBI_DMA1
#undef COALIBI_DMA2
#undef COALIBI_DMA4
#undef COALIBI_DMA_FIRST
#undef COALIBI_DMA_NEXT
#pragma clang diagnostic pop

// The source offsets of a wavefront's DMA of HALVES runs of 16 keys, the first of them half `half0` of its 32-key tile.
//   Lane ln of instruction m brings in piece ln % CPR of key m * KPI + ln / CPR.  The XOR patterns are linear in the key's
// bits, so their part that depends on m and on the half is a constant on top of the lane's own.
template <typename T, int D, bool V, int HALVES>
struct DmaOffsets {
  using C = TreeCfg<T, D>;
  int off[HALVES][C::HALF_INSTR];

  static constexpr __device__ __forceinline__ int pattern(int key) {
    return V ? swizzle_v<C::CPR, C::E>(key) : swizzle_k<C::CPR>(kRegOfRow(key));
  }
  __device__ __forceinline__ void init(int ld, int half0, int lane) {
    constexpr int KPI = 64 / C::CPR;  // keys per instruction
    const int key = lane / C::CPR & 15, piece = lane % C::CPR;
    const int row = key * (ld * C::E), own = (piece ^ pattern(key)) << 4, step = KPI * ld * C::E;
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      const int hx = (HALVES == 2 ? i : half0) * (pattern(16) << 4);
#pragma unroll
      for (int m = 0; m < C::HALF_INSTR; ++m) off[i][m] = row + m * step + (own ^ (pattern(m * KPI) << 4) ^ hx);
    }
  }
  // To LDS byte address lds.  Run i's rows start at base[i], rows[i] of them valid (the others land as zeros).
  template <bool NT>
  __device__ __forceinline__ void issue(const T* const (&base)[HALVES], const int (&rows)[HALVES], int ld, unsigned lds,
                                        int lane) const {
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      const __amdgpu_buffer_rsrc_t r = tile_rsrc(base[i], row_span(rows[i], ld, D));
      if (16 * C::ROWB >= 1024 || lane < C::ROWB) dma_run<C::HALF_INSTR, NT>(r, lds + 16 * i * C::ROWB, off[i]);
    }
  }
};

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

// WR: wavefronts over the query rows.  NT: the cache is read once (one row block), so its DMA does not keep it in L2.
template <typename T, int D, int WR, bool NT>
__global__ __launch_bounds__(kTreeThreads, (TreeCfg<T, D>::WGS_PER_CU)) void coalibi_tree_split_kernel(TreeArgs a) {
  using C = TreeCfg<T, D>;
  using M = Mfma<T>;
  using V8 = typename M::vec8;
  constexpr int WK = kTreeWaves / WR;             // wavefronts over the chunk's keys
  constexpr int NTILE = WR == 1 ? 1 : 2;          // 32-key tiles of a wavefront
  constexpr int CHUNK = tree_chunk_keys(32 * WR);  // keys
  constexpr int NBUF = kTreeLdsKeys / CHUNK;      // LDS buffers
  static_assert(CHUNK == WK * NTILE * kWaveKeys, "the wavefronts share out a chunk");
  constexpr int HALVES = CHUNK / kTreeWaves / 16;  // runs of 16 keys a wavefront brings in
  constexpr int INSTR = HALVES * C::HALF_INSTR;   // DMA instructions of its K (or V) of a chunk
  __shared__ __align__(1024) char smem[C::LDS_BYTES];
  __shared__ float sSig[2][WK][WR * 32];
  __shared__ float sMax[WK][WR * 32], sSum[WK][WR * 32], sScale[WK][WR * 32];
  __shared__ unsigned long long sBad;  // new keys whose values hold an infinity or a NaN
  __shared__ bool sLost[kTreeWaves];   // a wavefront found a filled row on no page of the pool

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane & 31, hh = lane >> 5;
  const int wr = wave % WR, wk = wave / WR;
  // Ids: the row blocks of an item (split, sequence, kv head) 8 apart, so that they share an XCD and its L2.
  const int RB = a.row_blocks, id = blockIdx.x;
  const int rb = (id >> 3) % RB, item = (id / (8 * RB)) * 8 + (id & 7);
  const int nS = a.nSplits;
  int cps = a.cps;
  TreeItem it{item / nS, item % nS};
  if (a.plan) {
    cps = plan_cps(a, lane);
    it = plan_item(a, cps, item, lane);
    if (it.bhk < 0) return;
  } else if (it.bhk >= a.B * a.Hkv) {
    return;
  }
  // Wave-uniform, which the divisions behind them hide from the compiler.
  const int bhk = __builtin_amdgcn_readfirstlane(it.bhk), split = __builtin_amdgcn_readfirstlane(it.split);
  const int b = __builtin_amdgcn_readfirstlane(bhk / a.Hkv), hkv = bhk - b * a.Hkv;
  const int L = __builtin_amdgcn_readfirstlane(filled_rows(a, b));
  const int chunks = __builtin_amdgcn_readfirstlane(chunks_of(a, L));
  TreeSplits sp = splits_of(a, cps, chunks);
  sp = {__builtin_amdgcn_readfirstlane(sp.cps), __builtin_amdgcn_readfirstlane(sp.used)};
  if (split >= sp.used) return;  // past this sequence's keys: the merge reads no such partial
  const bool newest = split == sp.used - 1;
  const int c_first = split * sp.cps, c_top = min(c_first + sp.cps, chunks) - 1;
  const int c_cache = chunks - 2;  // the newest chunk of filled rows; the one after it is the new keys

  const int R = a.G * a.T, row = rb * (WR * 32) + wr * 32 + hl;
  const bool row_ok = row < R;
  const int rsafe = row_ok ? row : 0;
  const int g = rsafe / a.T, t = rsafe - g * a.T, h = hkv * a.G + g;
  const float lam2 = a.slopes[h] * kLog2e;

  unsigned long long sees = 0;
  if (newest) {
    if (tid == 0 && nS > 1) a.used[bhk] = sp.used;  // every row block writes the same
    const unsigned long long all = ancestors(a, b, lane);
    sees = (unsigned long long)__shfl((unsigned)(all >> 32), t, 64) << 32 | __shfl((unsigned)all, t, 64);
    if (tid == 0) sBad = 0;
  }

  const T* const kn = head_at(static_cast<const T*>(a.k), a.kl, b, hkv);
  const T* const vn = head_at(static_cast<const T*>(a.v), a.vl, b, hkv);
  const T* const kc = static_cast<const T*>(a.kc) + (size_t)hkv * a.kcl.h;
  const T* const vc = static_cast<const T*>(a.vc) + (size_t)hkv * a.vcl.h;
  const unsigned ldsK = lds_address(smem), ldsV = ldsK + kTreeLdsKeys * C::ROWB;

  // This wavefront's keys of chunk c: the unit and the row in it of each run of 16.  `lost`: a filled row lies
  // on no page of the pool (such pages are read from unit 0).  A wavefront looks up only the keys it brings in, which every
  // wavefront's rows take part in: at the end its `lost` makes all rows of the work-group NaN.
  bool lost = false;
  struct Halves {
    int unit[HALVES], row[HALVES];
  };
  const int my_key = wave * (16 * HALVES);
  auto find = [&](int c) {
    Halves f;
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      const int r = c * CHUNK + my_key + 16 * i;
      f.unit[i] = b;
      f.row[i] = r;
      if (a.place.table != nullptr) {
        f.unit[i] = 0;
        f.row[i] = r & ((1 << a.place.page_shift) - 1);
        if (r < L) {
          const int u = scalar_load(a.place.table + (size_t)b * a.place.table_stride + (r >> a.place.page_shift));
          const bool in = u >= 0 && u < a.place.units;
          lost |= !in;
          f.unit[i] = in ? u : 0;
        }
      }
    }
    return f;
  };
  // This wavefront's part of chunk c's K or V into buffer `buf` (NT: the cache's rows; the new tokens' are read by every
  // row block).  The cache's source offsets are the same for every chunk.
  const int half0 = HALVES == 2 ? 0 : wave & 1;
  DmaOffsets<T, D, false, HALVES> k_off;
  DmaOffsets<T, D, true, HALVES> v_off;
  k_off.init(a.kcl.r, half0, lane);
  v_off.init(a.vcl.r, half0, lane);
  auto issue = [&](auto is_v, int c, const Halves& f, int buf) {
    constexpr bool V = decltype(is_v)::value;
    const unsigned lds = (V ? ldsV : ldsK) + (buf * CHUNK + my_key) * C::ROWB;
    const T* base[HALVES];
    int rows[HALVES];
    if (c > c_cache) {
      const int ld = V ? a.vl.r : a.kl.r;
#pragma unroll
      for (int i = 0; i < HALVES; ++i) {
        const int r = my_key + 16 * i;
        base[i] = (V ? vn : kn) + (size_t)r * ld;
        rows[i] = min(max(a.T - r, 0), 16);
      }
      DmaOffsets<T, D, V, HALVES> off;
      off.init(ld, half0, lane);
      off.template issue<false>(base, rows, ld, lds, lane);
    } else {
      const Layout& l = V ? a.vcl : a.kcl;
#pragma unroll
      for (int i = 0; i < HALVES; ++i) {
        base[i] = (V ? vc : kc) + (size_t)f.unit[i] * l.b + (size_t)f.row[i] * l.r;
        rows[i] = min(max(L - (c * CHUNK + my_key + 16 * i), 0), 16);
      }
      if constexpr (V)
        v_off.template issue<NT>(base, rows, l.r, lds, lane);
      else
        k_off.template issue<NT>(base, rows, l.r, lds, lane);
    }
  };
  using K_t = std::false_type;
  using V_t = std::true_type;

  // Q^T fragments: lane l holds query row l%32 of its tile (zero past R).
  V8 qf[C::KS];
  {
    const T* const q = head_at(static_cast<const T*>(a.q), a.ql, b, h) + (size_t)t * a.ql.r + hh * 8;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) qf[ks] = row_ok ? ld_vec8(q + ks * 16) : zero_vec8<T>();
  }
  Halves cur = c_top > c_cache ? Halves{} : find(c_top);
  issue(K_t{}, c_top, cur, 0);
  issue(V_t{}, c_top, cur, 0);
  // Wait here for Q: the compiler would place this wait inside the loop, as a vmcnt(0) of every chunk.
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));

  // State of the lane's row: scale (maximum, lazily followed), this half's share of the sum, O^T, and the sigma of
  // the keys after the current ones.
  float m2 = kNegInf, lsum = 0.f, carry = 0.f;
  f32x16 acc[C::DT];
#pragma unroll
  for (int j = 0; j < C::DT; ++j) acc[j] = f32x16{};

  // Lane constants of the operand reads.
  const int kx = swizzle_k<C::CPR>(hl);
  const char* const kread = smem + kRowOfReg(hl) * C::ROWB;
  const char* const vtile = smem + kTreeLdsKeys * C::ROWB;
  const int vi = lane & 15, vg = lane >> 4;
  const int tile0 = wk * NTILE;  // this wavefront's first 32-key tile of a chunk
  int par = 0, buf = 0;
  for (int c = c_top; c >= c_first; --c) {
    const bool more = c > c_first, fresh = c > c_cache;
    Halves next{};
    if (more) next = find(c - 1);
    if constexpr (NBUF == 2) {
      // This chunk has landed, and every wavefront has read the one before it, whose buffer the next one takes.
      wait_vm<0>();
      lds_barrier();
      if (more) {
        issue(K_t{}, c - 1, next, buf ^ 1);
        issue(V_t{}, c - 1, next, buf ^ 1);
      }
    } else {
      wait_vm<INSTR>();  // this chunk's K has landed once at most its V (issued after it) is outstanding
      if constexpr (WR > 1) lds_barrier();
    }
    const int key0 = c * CHUNK;
    {
      f32x16 sacc[NTILE];
#pragma unroll
      for (int st = 0; st < NTILE; ++st) sacc[st] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < C::KS; ++ks)
#pragma unroll
        for (int st = 0; st < NTILE; ++st) {
          const char* const kt = kread + (buf * CHUNK + (tile0 + st) * kWaveKeys) * C::ROWB;
          V8 kf;
          if constexpr (C::E == 2) {
            kf = *reinterpret_cast<const V8*>(kt + (((2 * ks + hh) ^ kx) << 4));
          } else {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(kt + (((4 * ks + 2 * hh) ^ kx) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(kt + (((4 * ks + 2 * hh + 1) ^ kx) << 4));
            kf = V8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          }
          sacc[st] = M::k16(kf, qf[ks], sacc[st]);
        }
      if (NBUF == 1 && more) {  // the K tiles have been read: the next chunk's come in
        wait_lds();
        if constexpr (WR > 1) lds_barrier();
        issue(K_t{}, c - 1, next, 0);
      }

      // Scores in log2 units; -inf for keys the row does not see: sigma 0, weight 0.  loc: the suffix sums of sigma
      // inside each lane's 16 keys.
      float loc[NTILE][16], tot[NTILE];
      const bool masked = fresh || key0 + (tile0 + NTILE) * kWaveKeys > L;
#pragma unroll
      for (int st = 0; st < NTILE; ++st) {
        const int kt = (tile0 + st) * kWaveKeys + 16 * hh;  // the lane's first key in the chunk
        if (masked) {
          const int left = L - key0 - kt;
          const unsigned ok = fresh ? (kt < 64 ? (unsigned)(sees >> (kt & 63)) : 0u)
                                    : left >= 16 ? 0xffffu : (1u << max(left, 0)) - 1u;
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[st][r] = ok >> r & 1 ? sacc[st][r] * a.sc2 : kNegInf;
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[st][r] *= a.sc2;
        }
        float run = 0.f;
#pragma unroll
        for (int r = 15; r >= 0; --r) {
          run += sigmoid_log2(sacc[st][r]);
          loc[st][r] = run;
        }
        tot[st] = run;
      }
      // off: the sigma after each lane's run.  Runs right to left: (tile 1, half 1), (1, 0), (0, 1), (0, 0).
      float off[NTILE], sum = 0.f;
#pragma unroll
      for (int st = NTILE - 1; st >= 0; --st) {
        const float oth = other_half(tot[st]);
        off[st] = sum + (hh ? 0.f : oth);
        sum += hh ? tot[st] + oth : oth + tot[st];
      }
      float after = carry;
      if constexpr (WK > 1) {
        if (hh == 0) sSig[par][wk][wr * 32 + hl] = sum;
        lds_barrier();  // the DMA in flight goes on
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float sw = sSig[par][w][wr * 32 + hl];
          after += w > wk ? sw : 0.f;
          carry += sw;
        }
        par ^= 1;
      } else {
        carry += sum;
      }

      // a relative to the row's scale is at most the largest score less cst, and the row's sum at least 1.  A chunk whose keys
      // all weigh less than 2^-a.far in every row of the wavefront is left out: its weights, and its V (a NaN or an
      // infinity among the scores or the sigmas keeps it).
      const float mb = m2 == kNegInf ? 0.f : m2;
      float cst[NTILE];
#pragma unroll
      for (int st = 0; st < NTILE; ++st) cst[st] = mb + lam2 * (after + off[st]);
      bool left_out = false;
      if constexpr (WR == 4) {
        bool near = row_ok && (fresh || m2 == kNegInf || !(lam2 >= 0.f));
#pragma unroll
        for (int st = 0; st < NTILE; ++st) {
          float mt = sacc[st][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) mt = fmaxf(mt, sacc[st][r]);
          near = near || (row_ok && (!(mt - cst[st] < -a.far) || !(tot[st] >= 0.f)));
        }
        left_out = !__any(near);
      }
      V8 pb[NTILE][2];
      if (!left_out) {
#pragma unroll
        for (int st = 0; st < NTILE; ++st)
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[st][r] = fmaf(-lam2, loc[st][r], sacc[st][r] - cst[st]);
        auto weights = [&] {
          float sum_p = 0.f;
#pragma unroll
          for (int st = 0; st < NTILE; ++st)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              f32x8 p;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                p[e] = fast_exp2(sacc[st][8 * s + e]);
                sum_p += p[e];  // before the rounding for the product: the LSE is fp32's
              }
              pb[st][s] = M::pack(p);
            }
          return sum_p;
        };
        float sum_p = weights();
        // The scale follows the maximum where the weights' sum says that it has risen far (or has none yet): no maximum is
        // taken otherwise.
        if (__any(m2 == kNegInf || sum_p > kTreeRescale)) {
          float mt = kNegInf;
#pragma unroll
          for (int st = 0; st < NTILE; ++st)
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sacc[st][r]);
          mt = fmaxf(mt, other_half(mt));
          const bool need = mt > (m2 == kNegInf ? kNegInf : 0.f);
          const float delta = need ? mt : 0.f;
          const float alpha = need ? (m2 == kNegInf ? 0.f : fast_exp2(-delta)) : 1.f;
          m2 = need ? mb + delta : m2;
          lsum *= alpha;
#pragma unroll
          for (int j = 0; j < C::DT; ++j) acc[j] *= alpha;
#pragma unroll
          for (int st = 0; st < NTILE; ++st) sacc[st] -= delta;
          sum_p = weights();
        }
        lsum += sum_p;
      }

      {
        if constexpr (NBUF == 1) {
          // This chunk's V has landed once at most the next chunk's K (issued by now) is outstanding.
          if (more)
            wait_vm<INSTR>();
          else
            wait_vm<0>();
          if constexpr (WR > 1) lds_barrier();
        }
        if (fresh) {
          // A product with a weight of 0 would carry an infinity or a NaN of a value to rows that do not see it: such
          // values become 0 here and are added to the rows that do below.
          char* const tile = smem + (kTreeLdsKeys + buf * CHUNK + my_key) * C::ROWB;
          for (int i = lane; i < 16 * HALVES * C::CPR; i += 64) {
            typedef T pieces __attribute__((ext_vector_type(16 / C::E)));
            pieces x = *reinterpret_cast<pieces*>(tile + i * 16);
            bool any = false;
#pragma unroll
            for (int e = 0; e < 16 / C::E; ++e)
              if (not_finite(static_cast<T>(x[e]))) {
                any = true;
                x[e] = T(0);
              }
            if (any) {
              *reinterpret_cast<pieces*>(tile + i * 16) = x;
              atomicOr(&sBad, 1ull << ((my_key + i / C::CPR) & 63));
            }
          }
          lds_barrier();
        }
      }
      // O^T[d][row] += V^T[d][key] P^T[key][row]; keys 8*s + 16*(l/32) + e of each tile, as in pb.
      if (!left_out)
#pragma unroll
      for (int st = 0; st < NTILE; ++st)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const char* const vt = vtile + (buf * CHUNK + (tile0 + st) * kWaveKeys) * C::ROWB;
#pragma unroll
          for (int j = 0; j < C::DT; ++j) {
            V8 va;
            if constexpr (C::E == 2) {
              const int r0 = 8 * s + (vg >> 1) * 16 + (vi >> 2), col = (32 * j + 16 * (vg & 1) + 4 * (vi & 3)) & (D - 1);
              const char* const at = vt + r0 * C::ROWB + (((col >> 3) ^ swizzle_v<C::CPR, 2>(vi >> 2)) << 4) + (col & 7) * 2;
              const u32x2 lo = lds_tr4(reinterpret_cast<const T*>(at));
              const u32x2 hi = lds_tr4(reinterpret_cast<const T*>(at + 4 * C::ROWB));
              va = __builtin_bit_cast(V8, u32x4{lo[0], lo[1], hi[0], hi[1]});
            } else {
              const int d = (32 * j + hl) & (D - 1);
              const char* const at = vt + (8 * s + 16 * hh) * C::ROWB + (((d >> 2) ^ swizzle_v<C::CPR, 4>(16 * hh)) << 4) + (d & 3) * 4;
#pragma unroll
              for (int e = 0; e < 8; ++e) va[e] = *reinterpret_cast<const float*>(at + e * C::ROWB);
            }
            acc[j] = M::k16(va, pb[st][s], acc[j]);
          }
        }
    }
    if (fresh) {
      unsigned long long bad = sBad;
      if (bad != 0) {
        for (int key = 0; key < a.T; ++key) {
          // The wavefront whose keys they are adds them (one of the WK), to rows that see the key.
          if (!(bad >> key & 1) || (WK > 1 && key / (kWaveKeys * NTILE) != wk) || !(sees >> key & 1)) continue;
#pragma unroll
          for (int j = 0; j < C::DT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = 32 * j + (r >> 2) * 8 + hh * 4 + (r & 3);
              if (d >= D) continue;
              const T x = vn[(size_t)key * a.vl.r + d];
              if (not_finite(x)) acc[j][r] += static_cast<float>(x);
            }
        }
      }
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    }
    if (NBUF == 1 && more) {
      wait_lds();  // the V tiles have been read
      if constexpr (WR > 1) lds_barrier();
      issue(V_t{}, c - 1, next, 0);
    }
    if constexpr (NBUF == 2) buf ^= 1;
  }

  // The row's sum over both halves, then over the wavefronts of its keys (in one z frame: the split's own keys).
  const float l = lsum + other_half(lsum);
  if (lane == 0) sLost[wave] = lost;
  const int rl = wr * 32 + hl;
  if (hh == 0) {
    sMax[wk][rl] = m2;
    sSum[wk][rl] = l;
  }
  __syncthreads();  // and every wavefront is done with the tiles (no DMA in flight)
  if (tid < WR * 32) {
    float m = kNegInf;
#pragma unroll
    for (int w = 0; w < WK; ++w) m = fmaxf(m, sMax[w][tid]);
    float ls = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float f = sMax[w][tid] == kNegInf ? 0.f : fast_exp2(sMax[w][tid] - m);
      sScale[w][tid] = f;
      ls += sMax[w][tid] == kNegInf && sSum[w][tid] == 0.f ? 0.f : f * sSum[w][tid];
    }
    bool any_lost = false;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) any_lost |= sLost[w];
    sMax[0][tid] = m;
    sSum[0][tid] = any_lost ? __builtin_nanf("") : ls;
  }
  __syncthreads();
  float* const so = reinterpret_cast<float*>(smem) + (size_t)(wk * WR + wr) * 32 * C::LDO;
  const float f = sScale[wk][rl];
#pragma unroll
  for (int j = 0; j < C::DT; ++j)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = 32 * j + q4 * 8 + hh * 4;
      if (d < D)
        *reinterpret_cast<f32x4*>(so + hl * C::LDO + d) =
            f32x4{acc[j][4 * q4] * f, acc[j][4 * q4 + 1] * f, acc[j][4 * q4 + 2] * f, acc[j][4 * q4 + 3] * f};
    }
  const size_t row0 = (size_t)bhk * R + rb * (WR * 32);  // the block's first row in o, lse and the partials
  const int rows = min(R - rb * (WR * 32), WR * 32);
  const bool direct = sp.used == 1;  // the whole sequence: no partials, and the merge leaves its rows alone
  if (wk == 0 && hh == 0 && row_ok) {
    const bool absent = newest && sees == 0;
    if (direct) {
      const float ls = sSum[0][rl];
      if (a.lse != nullptr) a.lse[row0 + rl] = absent ? kNegInf : (sMax[0][rl] + log2f(ls)) * kLn2;
      sScale[0][rl] = absent ? 0.f : 1.f / ls;
      sMax[0][rl] = absent ? 0.f : 1.f;
    } else {
      const size_t pi = (row0 + rl) * nS + split;
      a.pmax[pi] = sMax[0][rl];
      a.psum[pi] = absent ? kAbsent : sSum[0][rl];
      a.psig[pi] = carry;
    }
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += kTreeThreads) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    f32x4 s = f32x4{};
#pragma unroll
    for (int w = 0; w < WK; ++w)
      s += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(smem) + ((size_t)w * WR * 32 + r) * C::LDO + d);
    if (direct) {
      typedef T out4 __attribute__((ext_vector_type(4)));
      const bool there = sMax[0][r] != 0.f;
      const float inv = sScale[0][r];
      out4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(there ? s[e] * inv : 0.f);
      *reinterpret_cast<out4*>(static_cast<T*>(a.o) + (row0 + r) * D + d) = v;
    } else {
      *reinterpret_cast<f32x4*>(a.pout + ((row0 + r) * nS + split) * D + d) = s;
    }
  }
}

constexpr int kTreeMergeThreads = 256;

// O and LSE of a query row from its split partials: WPR wavefronts per row (one where rows are many, four where
// few rows have many splits each).
template <typename T, int D, int WPR>
__global__ __launch_bounds__(kTreeMergeThreads) void coalibi_tree_merge_kernel(TreeArgs a) {
  constexpr int ROWS = kTreeMergeThreads / 64 / WPR;  // rows per work-group
  constexpr int LPS = D / 4;                          // lanes per split's O
  constexpr int PER = 64 / LPS;                       // splits per wavefront and load
  __shared__ float sW[kTreeMergeThreads / 64][kMaxTreeSplits];
  __shared__ __align__(16) float sO[kTreeMergeThreads / 64][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = wave % WPR;
  const long long total = (long long)a.B * a.Hq * a.T;
  const long long mine = (long long)blockIdx.x * ROWS + wave / WPR;
  const long long row = mine < total ? mine : total - 1;  // every wavefront meets the barrier
  const int bh = (int)(row / a.T), b = bh / a.Hq;
  const float lam2 = a.slopes[bh - b * a.Hq] * kLog2e;
  const float* const pmax = a.pmax + row * a.nSplits;
  const float* const psum = a.psum + row * a.nSplits;
  const float* const psig = a.psig + row * a.nSplits;
  float* const w = sW[wave];
  // The usual split counts' statistics, read along with the count itself.
  const bool pre = lane < a.nSplits;
  const float sig0 = pre ? psig[lane] : 0.f, max0 = pre ? pmax[lane] : 0.f, sum0 = pre ? psum[lane] : 0.f;
  const int n = a.used[bh / a.G];  // the splits that wrote a partial
  if (WPR > 1 && n == 1) return;   // its only split wrote o (one row per work-group: nobody is left at a barrier)
  const bool absent = n <= 64 ? __shfl(sum0, n - 1, 64) == kAbsent : psum[n - 1] == kAbsent;

  // Split maxima shifted by the sigma of the splits after them; each wavefront computes all of them.
  float carry = 0.f, mx = kNegInf;
  for (int base = (n - 1) / 64 * 64; base >= 0; base -= 64) {
    const int s = base + lane;
    const bool ok = s < n;
    const float x = !ok ? 0.f : base == 0 ? sig0 : psig[s], pm = !ok ? kNegInf : base == 0 ? max0 : pmax[s];
    float suf = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const float y = __shfl_down(suf, off, 64);
      if (lane + off < 64) suf += y;
    }
    const float m = pm - lam2 * (carry + (suf - x));
    if (ok) w[s] = m;
    mx = fmaxf(mx, m);
    carry += __shfl(suf, 0, 64);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  const float mref = mx == kNegInf ? 0.f : mx;
  const float cut = __builtin_isinf(a.far) ? 0.f : 0x1p-64f;
  float l = 0.f;
  for (int s = lane; s < n; s += 64) {  // a lane reads back what it wrote itself
    const float f = fast_exp2(w[s] - mref), sum = s == lane ? sum0 : psum[s];
    // A split's O is not read where its weights' sum, and with it each of its keys' weights, is below 2^-64 of the row's
    // (which is at least 1 here): on a steep head all but the newest ones.  (The fp32 tail skip's bound; without the tail
    // skip all are read.  f alone would not do: a key may weigh kTreeRescale times its split's scale.)  The newest split holds
    // the new keys, which always count.
    w[s] = s < n - 1 && f * sum < cut ? -1.f : f;
    l = fmaf(f, sum, l);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
  wait_lds();  // the weights are read across lanes below (LDS operations of a wavefront complete in order)

  const int sub = lane / LPS, d = (lane % LPS) * 4;
  const float* const po = a.pout + row * a.nSplits * D + d;
  f32x4 acc[4] = {};
  constexpr int STRIDE = PER * WPR;
  for (int s = n - 1 - (part * PER + sub); s >= 0; s -= 4 * STRIDE) {
    f32x4 x[4];
    float f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = s - u * STRIDE;
      f[u] = at >= 0 ? w[at] : -1.f;
      x[u] = !(f[u] < 0.f) ? *reinterpret_cast<const f32x4*>(po + (size_t)at * D) : f32x4{};  // NaN is read, too
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] += f[u] * x[u];
  }
  f32x4 o = (acc[0] + acc[1]) + (acc[2] + acc[3]);
#pragma unroll
  for (int off = LPS; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off, 64);
  if constexpr (WPR > 1) {
    if (sub == 0) *reinterpret_cast<f32x4*>(&sO[wave][d]) = o;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int p = 1; p < WPR; ++p) o += *reinterpret_cast<const f32x4*>(&sO[wave + p][d]);
  }
  if (mine >= total || n == 1) return;
  if (sub == 0) {
    typedef T out4 __attribute__((ext_vector_type(4)));
    const float inv = 1.f / l;
    out4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(absent ? 0.f : o[e] * inv);
    *reinterpret_cast<out4*>(static_cast<T*>(a.o) + row * D + d) = v;
  }
  if (part == 0 && lane == 0 && a.lse != nullptr) a.lse[row] = absent ? kNegInf : (mx + log2f(l)) * kLn2;
}

template <typename T, int D, int WR>
hipError_t launch_split(const TreeArgs& a, hipStream_t stream) {
  // Under a plan at most one round of work-groups and a rounded-up split per sequence.
  const long long even = (long long)a.B * a.Hkv * a.nSplits;
  const long long items = a.plan ? std::min<long long>(even, ((long long)a.share + a.B) * a.Hkv) : even;
  const dim3 grid(static_cast<unsigned>((items + 7) / 8 * 8 * a.row_blocks));
  if (a.row_blocks == 1)
    hipLaunchKernelGGL((coalibi_tree_split_kernel<T, D, WR, true>), grid, dim3(kTreeThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((coalibi_tree_split_kernel<T, D, WR, false>), grid, dim3(kTreeThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

template <typename T, int D>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int R = a.G * a.T;
  hipError_t e;
  if (R <= 32)
    e = launch_split<T, D, 1>(a, stream);
  else if (R <= 64)
    e = launch_split<T, D, 2>(a, stream);
  else
    e = launch_split<T, D, 4>(a, stream);
  if (e != hipSuccess || a.nSplits == 1) return e;
  const long long rows = (long long)a.B * a.Hq * a.T;
  // Four wavefronts a row against one, whole step in us at D 128: 128 rows 31.5 against 33.3, 512 rows 37.0 against 38.7,
  // 2048 rows 39.0 against 37.1 (and 62.6 against 61.7), 12288 rows 135 against 124.
  if (rows <= 1024)
    hipLaunchKernelGGL((coalibi_tree_merge_kernel<T, D, 4>), dim3(static_cast<unsigned>(rows)), dim3(kTreeMergeThreads), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((coalibi_tree_merge_kernel<T, D, 1>), dim3(static_cast<unsigned>((rows + 3) / 4)),
                       dim3(kTreeMergeThreads), 0, stream, a);
  return hipGetLastError();
}

#define COALIBI_INST_TREE(T, D) template hipError_t launch_tree<T, D>(const TreeArgs&, hipStream_t);
COALIBI_INST_TREE(_Float16, 16)
COALIBI_INST_TREE(_Float16, 32)
COALIBI_INST_TREE(_Float16, 64)
COALIBI_INST_TREE(_Float16, 128)
COALIBI_INST_TREE(_Float16, 256)
COALIBI_INST_TREE(__bf16, 16)
COALIBI_INST_TREE(__bf16, 32)
COALIBI_INST_TREE(__bf16, 64)
COALIBI_INST_TREE(__bf16, 128)
COALIBI_INST_TREE(__bf16, 256)
COALIBI_INST_TREE(float, 16)
COALIBI_INST_TREE(float, 32)
COALIBI_INST_TREE(float, 64)
COALIBI_INST_TREE(float, 128)

}  // namespace coalibi
