// Appending keys and values to a cache (paged, or one contiguous cache per sequence) on gfx950.
//
// Row i of sequence b -- the new row rows[b][i], or i -- is copied to cache row seq_lens[b] + i of every kv
// head, for i < counts[b].  A copy of 2 * rows * D elements in and out, bound by HBM for prompts and by the
// launch for single tokens: one thread per 16-byte chunk, so that a wavefront's loads and stores are
// runs of whole rows, and K and V in one launch.  Captured: 1 row for each of 16 sequences 2.4 us (an empty kernel 2.1),
// 8 prompts of up to 2048 rows, 80 MB, 17.9 us (a large copy's rate gives 15.8).
//
// Rows that have no place are left out: counts past N or below 0 are clamped, a source row outside [0, T), a
// cache row outside [0, capacity) and a table entry outside the pool write nothing.
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

constexpr int kAppendThreads = 256;

// The element offset of a cache row, or -1 where it has no place.
__device__ __forceinline__ long long cache_row(const CachePlace& p, const Layout& l, int b, int h, int row) {
  int unit = b;
  if (p.table != nullptr) {
    unit = p.table[(size_t)b * p.table_stride + (row >> p.page_shift)];
    if (unit < 0 || unit >= p.units) return -1;
    row &= (1 << p.page_shift) - 1;
  }
  return (long long)unit * l.b + (long long)h * l.h + (long long)row * l.r;
}

__global__ __launch_bounds__(kAppendThreads) void coalibi_append_kernel(AppendArgs a) {
  const int per_row = a.row_chunks;
  const long long per_seq = (long long)a.N * a.Hkv * per_row;
  const long long at = (long long)blockIdx.x * kAppendThreads + threadIdx.x;
  if (at >= per_seq) return;
  const int c = (int)(at % per_row);
  const int hi = (int)(at / per_row);  // (i, h), heads fastest: at most 2^31 by the host's check
  const int i = hi / a.Hkv, h = hi - i * a.Hkv;
  const bool value = blockIdx.z != 0;
  const Layout& from = value ? a.vl : a.kl;
  const Layout& to = value ? a.vcl : a.kcl;
  const char* const src = static_cast<const char*>(value ? a.v : a.k);
  char* const dst = static_cast<char*>(value ? a.vc : a.kc);
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    if (a.counts != nullptr && i >= a.counts[b]) continue;
    const int row = a.rows == nullptr ? i : a.rows[(size_t)b * a.N + i];
    const long long pos = (long long)a.seq_lens[b] + i;
    if (row < 0 || row >= a.T || pos < 0 || pos >= a.capacity) continue;
    const long long off = cache_row(a.place, to, b, h, (int)pos);
    if (off < 0) continue;
    const long long s = (long long)b * from.b + (long long)h * from.h + (long long)row * from.r;
    *reinterpret_cast<uint4*>(dst + off * a.elem + c * 16) = *reinterpret_cast<const uint4*>(src + s * a.elem + c * 16);
  }
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t stream) {
  const long long per_seq = (long long)a.N * a.Hkv * a.row_chunks;
  const dim3 grid(static_cast<unsigned>((per_seq + kAppendThreads - 1) / kAppendThreads),
                  static_cast<unsigned>(std::min(a.B, 65535)), 2);
  hipLaunchKernelGGL(coalibi_append_kernel, grid, dim3(kAppendThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace coalibi
