// Co-ALiBi attention of a step's new tokens -- one token, a run of them or a tree of drafts -- over a key /
// value cache and each other, on gfx950.
//
// Node t of a sequence sees the cache's filled rows and, after them, its chain of ancestors up to itself.
// Parents come before their children, so those of the T new keys that a node sees stand in index order
// and are the bits of a 64-bit mask.  With the keys in this order, as in the decode (coalibi_decode.hip):
//   t_j = sm_scale*log2(e) * q.k_j,   sigma_j = sigmoid(t_j / log2(e)),
//   z_j = sum_{k >= j} sigma_k,       a_j = t_j - slope*log2(e) * z_j,
//   O   = sum_j 2^(a_j - m) v_j / sum_j 2^(a_j - m),   LSE = (m + log2 l) * ln 2.
#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

constexpr int kTreeThreads = 256;

__device__ __forceinline__ int filled_rows(const TreeArgs& a, int b) {
  return a.seq_lens == nullptr ? a.L : min(max(a.seq_lens[b], 0), a.L);
}

// The new keys node t sees (bit j: key j), or 0 for an absent node: one whose chain of parents leaves
// [-1, own index).
__device__ __forceinline__ unsigned long long ancestors(const TreeArgs& a, int b, int t) {
  if (a.parents == nullptr) return t == 63 ? ~0ull : (2ull << t) - 1;
  const int* par = a.parents + (size_t)b * a.parents_stride;
  unsigned long long m = 0;
  while (t >= 0) {
    m |= 1ull << t;
    const int p = par[t];
    if (p < -1 || p >= t) return 0;
    t = p;
  }
  return m;
}

template <typename F>
__device__ __forceinline__ float block_reduce(float x, float* red, const F& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int off = 32; off > 0; off >>= 1) x = f(x, __shfl_xor(x, off, 64));
  if (lane == 0) red[wave] = x;
  __syncthreads();
  x = red[0];
  for (int w = 1; w < kTreeThreads / 64; ++w) x = f(x, red[w]);
  __syncthreads();
  return x;
}

// One work-group per (batch, query head, node), its keys 256 at a time from the newest on.
template <typename T>
__global__ __launch_bounds__(kTreeThreads) void coalibi_tree_kernel(TreeArgs a) {
  __shared__ float sq[256], sp[kTreeThreads], red[kTreeThreads / 64];
  __shared__ const T* srow[kTreeThreads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int id = blockIdx.x, t = id % a.T, h = id / a.T % a.Hq, b = id / a.T / a.Hq, hkv = h / a.G;
  const float lam2 = a.slopes[h] * kLog2e;
  const int L = filled_rows(a, b);
  const unsigned long long sees = ancestors(a, b, t);
  T* const orow = static_cast<T*>(a.o) + (size_t)id * a.D;
  if (sees == 0) {
    for (int d = tid; d < a.D; d += kTreeThreads) orow[d] = T(0);
    if (tid == 0 && a.lse != nullptr) a.lse[id] = kNegInf;
    return;
  }
  const T* const q = head_at(static_cast<const T*>(a.q), a.ql, b, h) + (size_t)t * a.ql.r;
  if (tid < a.D) sq[tid] = static_cast<float>(q[tid]);
  __syncthreads();
  const T* const knew = head_at(static_cast<const T*>(a.k), a.kl, b, hkv);
  const T* const vnew = head_at(static_cast<const T*>(a.v), a.vl, b, hkv);
  float m = kNegInf, l = 0.f, carry = 0.f, acc = 0.f;
  bool lost = false;  // a visible row lies on no page of the pool
  // Step -1: the new tokens; then the cache's rows from its end on.
  for (int k0 = -1; k0 == -1 || k0 * kTreeThreads < L; ++k0) {
    const int j = k0 < 0 ? tid : L - 1 - k0 * kTreeThreads - (kTreeThreads - 1 - tid);
    const bool ok = k0 < 0 ? tid < a.T && (sees >> tid & 1) : j >= 0;
    float s = kNegInf, sig = 0.f;
    const T* vrow = nullptr;
    if (ok) {
      const T* krow;
      if (k0 < 0) {
        krow = knew + (size_t)j * a.kl.r;
        vrow = vnew + (size_t)j * a.vl.r;
      } else {
        int unit = b, r = j;
        if (a.place.table != nullptr) {
          unit = a.place.table[(size_t)b * a.place.table_stride + (j >> a.place.page_shift)];
          r = j & ((1 << a.place.page_shift) - 1);
          if (unit < 0 || unit >= a.place.units) lost = true, unit = 0;
        }
        krow = head_at(static_cast<const T*>(a.kc), a.kcl, unit, hkv) + (size_t)r * a.kcl.r;
        vrow = head_at(static_cast<const T*>(a.vc), a.vcl, unit, hkv) + (size_t)r * a.vcl.r;
      }
      s = 0.f;
      for (int d = 0; d < a.D; ++d) s += sq[d] * static_cast<float>(krow[d]);
      s *= a.sc2;
      sig = sigmoid_log2(s);
    }
    srow[tid] = vrow;
    float suf = sig;  // suffix sum over the block
    for (int off = 1; off < 64; off <<= 1) {
      const float y = __shfl_down(suf, off, 64);
      if (lane + off < 64) suf += y;
    }
    if (lane == 0) red[wave] = suf;
    __syncthreads();
    float after = carry, all = 0.f;
    for (int w = 0; w < kTreeThreads / 64; ++w) {
      if (w > wave) after += red[w];
      all += red[w];
    }
    __syncthreads();
    const float av = ok ? s - lam2 * (after + suf) : kNegInf;
    carry += all;
    const float mt = block_reduce(av, red, [](float x, float y) { return fmaxf(x, y); });
    const float mn = fmaxf(m, mt), mref = mn == kNegInf ? 0.f : mn;
    const float p = fast_exp2(av - mref), fold = fast_exp2(m - mref);
    m = mn;
    l = l * fold + block_reduce(p, red, [](float x, float y) { return x + y; });
    sp[tid] = p;
    __syncthreads();
    acc *= fold;
    if (tid < a.D)
      for (int e = 0; e < kTreeThreads; ++e)
        if (srow[e] != nullptr) acc += sp[e] * static_cast<float>(srow[e][tid]);
    __syncthreads();
  }
  if (__syncthreads_or(lost)) l = __builtin_nanf("");
  if (tid < a.D) orow[tid] = static_cast<T>(acc / l);
  if (tid == 0 && a.lse != nullptr) a.lse[id] = (m + log2f(l)) * kLn2;
}

}  // namespace

template <typename T>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.B) * a.Hq * a.T);
  hipLaunchKernelGGL((coalibi_tree_kernel<T>), grid, dim3(kTreeThreads), 0, stream, a);
  return hipGetLastError();
}

template hipError_t launch_tree<_Float16>(const TreeArgs&, hipStream_t);
template hipError_t launch_tree<__bf16>(const TreeArgs&, hipStream_t);
template hipError_t launch_tree<float>(const TreeArgs&, hipStream_t);

}  // namespace coalibi
