// Beam search on gfx950: the best continuations over a sequence's beams and the vocabulary, and the paged cache that follows
// them.
//
// Selection: with M_w and S_w a row's largest logit and sum_t exp(x_t - M_w), candidate (w, t) scores
//   score_w + (x_t - M_w) - log S_w.
// Within a row the order is the logits', so that each segment of a row yields its maximum, its sum and its N largest logits in
// one read (its elements stay in registers), and a second launch ranks those of a sequence's beams.  Exponentials are fp32's,
// summed in fp64 over the threads; scores are fp64 until they are written.
//   The N largest of a segment: the N-th largest of the 256 threads' maxima is at most the N-th largest element, and few others
// are above it.  Those at or above it are listed and ranked by counting.  Where equal logits make the list overflow, N rounds
// of a search for the next one take its place.
//
// Reordering: a group of W beams owns W pages in every column of its block table.  Pages that are full are shared by all that
// descend from them; one in use stays with the first of its heirs, and the others get free pages of its column and copies of
// its rows.  That many are free, as no more than W are in use.  Every wavefront works out its column's W beams by itself, a lane
// each, so that tables and copies are one launch.
#include <algorithm>

#include "coalibi_common.h"
#include "coalibi_kernels.h"

namespace coalibi {

namespace {

constexpr int kSelectThreads = 256;
constexpr int kListed = 1024;  // candidates of a list that are ranked by counting

__device__ __forceinline__ bool better(float xa, int ia, float xb, int ib) { return xa > xb || (xa == xb && ia < ib); }

// The best of the work-group's (value, place) pairs, in every thread; a place below 0 is none.
template <typename X, typename Better>
__device__ __forceinline__ void best_of_block(X& x, int& at, X* sx, int* si, Better better) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const X ox = __shfl_xor(x, off, 64);
    const int oi = __shfl_xor(at, off, 64);
    if (oi >= 0 && (at < 0 || better(ox, oi, x, at))) {
      x = ox;
      at = oi;
    }
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sx[threadIdx.x >> 6] = x;
    si[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  for (int w = 0; w < kSelectThreads / 64; ++w)
    if (si[w] >= 0 && (at < 0 || better(sx[w], si[w], x, at))) {
      x = sx[w];
      at = si[w];
    }
}

// E: elements of a segment per thread.
template <typename T, int E>
__global__ __launch_bounds__(kSelectThreads) void coalibi_select_rows_kernel(SelectArgs a) {
  __shared__ float sx[kListed];
  __shared__ int si[kListed];
  __shared__ float wx[kSelectThreads / 64];
  __shared__ int wi[kSelectThreads / 64];
  __shared__ double ws[kSelectThreads / 64];
  __shared__ int count;
  __shared__ float cut;
  const int tid = threadIdx.x, seg = blockIdx.x;
  const long long row = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  if (row >= (long long)a.B * a.W) return;
  if (a.finished != nullptr && a.finished[row] != 0) return;
  const int b = (int)(row / a.W), w = (int)(row - (long long)b * a.W);
  const T* const x = static_cast<const T*>(a.logits) + (size_t)b * a.batch_stride + (size_t)w * a.beam_stride;
  const int first = seg * a.per_segment, n = min(a.V - first, a.per_segment);
  float v[E];
  bool nan = false;
  float top = kNegInf;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = tid + e * kSelectThreads;
    v[e] = i < n ? static_cast<float>(x[first + i]) : kNegInf;
    nan |= v[e] != v[e];
    top = fmaxf(top, v[e]);
  }
  const size_t part = (size_t)row * a.segments + seg;
  float* const oval = a.pval + part * a.N;
  int* const otok = a.ptok + part * a.N;
  // The segment's maximum (a NaN: none), then its sum.
  float m = top;
  int at = __any(nan) ? -1 : tid;
  {
    // A wavefront with a NaN says so by a place below 0.
    float wm = m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) wm = fmaxf(wm, __shfl_xor(wm, off, 64));
    if ((tid & 63) == 0) {
      wx[tid >> 6] = wm;
      wi[tid >> 6] = at;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    m = wx[0];
    for (int i = 1; i < kSelectThreads / 64; ++i) m = fmaxf(m, wx[i]);
    nan = false;
    for (int i = 0; i < kSelectThreads / 64; ++i) nan |= wi[i] < 0;
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) sum += v[e] == m ? (m == kNegInf ? 0.f : 1.f) : fast_exp2((v[e] - m) * kLog2e);
  double total = sum;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if ((tid & 63) == 0) ws[tid >> 6] = total;
  sx[tid] = top;
  __syncthreads();
  if (tid == 0) {
    a.pmax[part] = nan ? __builtin_nanf("") : m;
    a.psum[part] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
  }
  if (nan) return;
  // The N-th largest of the threads' maxima.
  {
    int rank = 0;
    for (int i = 0; i < kSelectThreads; i += 4) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(sx + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) rank += y[e] > top || (y[e] == top && i + e < tid) ? 1 : 0;
    }
    if (rank == a.N - 1) cut = top;
  }
  __syncthreads();
  const float least = cut;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (v[e] >= least && v[e] > kNegInf) {
      const int p = atomicAdd(&count, 1);
      if (p < kListed) {
        sx[p] = v[e];
        si[p] = first + tid + e * kSelectThreads;
      }
    }
  __syncthreads();
  const int c = count;
  if (c <= kListed) {
    for (int i = tid; i < c; i += kSelectThreads) {
      const float xi = sx[i];
      const int ti = si[i];
      int rank = 0;
      for (int j = 0; j < c; ++j) rank += better(sx[j], si[j], xi, ti) ? 1 : 0;
      if (rank < a.N) {
        oval[rank] = xi;
        otok[rank] = ti;
      }
    }
    for (int i = c + tid; i < a.N; i += kSelectThreads) otok[i] = -1;
  } else {
    float last = __builtin_inff();
    int last_at = -1;
    for (int k = 0; k < a.N; ++k) {
      float best = kNegInf;
      int best_at = -1;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = first + tid + e * kSelectThreads;
        if (v[e] > kNegInf && (k == 0 || better(last, last_at, v[e], i)) && (best_at < 0 || better(v[e], i, best, best_at))) {
          best = v[e];
          best_at = i;
        }
      }
      best_of_block(best, best_at, wx, wi, [](float xa, int ia, float xb, int ib) { return better(xa, ia, xb, ib); });
      last = best;
      last_at = best_at;
      if (tid == 0) {
        oval[k] = best;
        otok[k] = best_at;
      }
      if (best_at < 0) {  // fewer than N logits above -inf
        for (int i = k + 1 + tid; i < a.N; i += kSelectThreads) otok[i] = -1;
        break;
      }
    }
  }
}

// The N best of a sequence's candidates, which stand in the order (beam, segment, rank).
__global__ __launch_bounds__(kSelectThreads) void coalibi_select_beams_kernel(SelectArgs a) {
  __shared__ double sbase[kMaxBeams];  // score - log S, or NaN for a beam without candidates
  __shared__ float smax[kMaxBeams];
  __shared__ double sx[kListed];
  __shared__ int si[kListed];
  __shared__ double cut;
  __shared__ int cut_at, count;
  __shared__ double wx[kSelectThreads / 64];
  __shared__ int wi[kSelectThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const long long row0 = (long long)b * a.W;
  const int per_beam = a.segments * a.N, total = a.W * per_beam;
  if (tid == 0) {
    count = 0;
    cut_at = -1;
  }
  for (int w = wave; w < a.W; w += kSelectThreads / 64) {
    const long long row = row0 + w;
    const float score = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    double base = done ? (double)score : __builtin_nan("");
    float m = 0.f;
    if (!done) {
      const float* const pm = a.pmax + row * a.segments;
      const double* const ps = a.psum + row * a.segments;
      bool nan = false;
      m = kNegInf;
      for (int s = lane; s < a.segments; s += 64) {
        nan |= pm[s] != pm[s];
        m = fmaxf(m, pm[s]);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
      double sum = 0.0;
      for (int s = lane; s < a.segments; s += 64) sum += pm[s] == m ? ps[s] : ps[s] * exp((double)pm[s] - (double)m);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      if (!__any(nan) && m > kNegInf) base = (double)score - log(sum);
    }
    if (lane == 0) {
      sbase[w] = score > kNegInf && score < __builtin_inff() ? base : __builtin_nan("");
      smax[w] = m;
    }
  }
  __syncthreads();
  // Candidate i: its score, NaN for none.
  auto candidate = [&](int i) -> double {
    const int w = i / per_beam, k = i - w * per_beam;
    const double base = sbase[w];
    if (base != base) return base;
    if (a.finished != nullptr && a.finished[row0 + w] != 0) return k == 0 ? base : __builtin_nan("");
    const size_t at = (size_t)(row0 + w) * per_beam + k;
    if (a.ptok[at] < 0) return __builtin_nan("");
    const float x = a.pval[at], m = smax[w];
    // Of +inf logits all weigh 1, and every other one nothing.
    return x == m ? base : m == __builtin_inff() ? __builtin_nan("") : base + ((double)x - (double)m);
  };
  // Equal scores go by beam, then by logit, then by token.  (Logits that differ may score the same in 64 bits, where they are
  // far smaller than the row's largest.)
  auto better = [&](double xa, int ia, double xb, int ib) {
    if (xa != xb) return xa > xb;
    const int wa = ia / per_beam, wb = ib / per_beam;
    if (wa != wb || ia == ib || (a.finished != nullptr && a.finished[row0 + wa] != 0)) return ia < ib;
    const size_t pa = (size_t)row0 * per_beam + ia, pb = (size_t)row0 * per_beam + ib;
    return a.pval[pa] > a.pval[pb] || (a.pval[pa] == a.pval[pb] && a.ptok[pa] < a.ptok[pb]);
  };
  // As for the segments: the N-th best of the threads' best ones bounds what can be selected.
  double best = 0.0;
  int best_at = -1;
  for (int i = tid; i < total; i += kSelectThreads) {
    const double x = candidate(i);
    if (x == x && (best_at < 0 || better(x, i, best, best_at))) {
      best = x;
      best_at = i;
    }
  }
  sx[tid] = best;
  si[tid] = best_at;
  __syncthreads();
  if (best_at >= 0) {
    int rank = 0;
    for (int j = 0; j < kSelectThreads; ++j) rank += si[j] >= 0 && better(sx[j], si[j], best, best_at) ? 1 : 0;
    if (rank == a.N - 1) {
      cut = best;
      cut_at = best_at;
    }
  }
  __syncthreads();
  const double least = cut;
  const int least_at = cut_at;  // below 0: fewer than N threads have any, and all are listed
  for (int i = tid; i < total; i += kSelectThreads) {
    const double x = candidate(i);
    if (x == x && (least_at < 0 || !better(least, least_at, x, i))) {
      const int p = atomicAdd(&count, 1);
      if (p < kListed) {
        sx[p] = x;
        si[p] = i;
      }
    }
  }
  __syncthreads();
  const int c = count;
  auto write = [&](int k, double x, int i) {
    const int w = i < 0 ? 0 : i / per_beam;
    const size_t o = (size_t)b * a.N + k;
    a.out_scores[o] = i < 0 ? kNegInf : (float)x;
    a.out_parents[o] = w;
    a.out_tokens[o] = i < 0 ? -1
                      : a.finished != nullptr && a.finished[row0 + w] != 0
                          ? a.end_token
                          : a.ptok[(size_t)(row0 + w) * per_beam + (i - w * per_beam)];
  };
  if (c <= kListed) {
    for (int i = tid; i < c; i += kSelectThreads) {
      const double xi = sx[i];
      const int ti = si[i];
      int rank = 0;
      for (int j = 0; j < c; ++j) rank += better(sx[j], si[j], xi, ti) ? 1 : 0;
      if (rank < a.N) write(rank, xi, ti);
    }
    for (int i = c + tid; i < a.N; i += kSelectThreads) write(i, 0.0, -1);
  } else {
    double last = 0.0;
    int last_at = -1;
    for (int k = 0; k < a.N; ++k) {
      double x = 0.0;
      int at = -1;
      for (int i = tid; i < total; i += kSelectThreads) {
        const double y = candidate(i);
        if (y == y && (k == 0 || better(last, last_at, y, i)) && (at < 0 || better(y, i, x, at))) {
          x = y;
          at = i;
        }
      }
      best_of_block(x, at, wx, wi, better);
      last = x;
      last_at = at;
      if (tid == 0) write(k, x, at);
    }
  }
}

// What becomes of a group's pages in one column; lane i is beam i.
struct Column {
  int from, to;  // the parent's page, the beam's
  int rows;      // filled rows of it, all of which `to` has to get where it is another page
  int len;
  bool copies;
};
__device__ __forceinline__ Column column(const ReorderArgs& a, int g, int j, int lane, int* free_pages) {
  const bool is = lane < a.W;
  const size_t mine = (size_t)g * a.W + (is ? lane : 0);
  const int par = min(max(a.parents[mine], 0), a.W - 1);
  const size_t of = (size_t)g * a.W + par;
  Column c;
  c.len = a.lens[of];
  c.from = a.table[of * a.J + j];
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

__global__ __launch_bounds__(kReorderThreads) void coalibi_reorder_kernel(ReorderArgs a) {
  __shared__ int sfree[kReorderThreads / 64][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int beams = a.B * a.W;
  if (blockIdx.y == (unsigned)a.pools) {  // the tables: a wavefront per group and column
    const long long columns = (long long)a.B * a.J;
    for (long long at = (long long)blockIdx.x * (kReorderThreads / 64) + wave; at < columns;
         at += (long long)gridDim.x * (kReorderThreads / 64)) {
      const int g = (int)(at / a.J), j = (int)(at - (long long)g * a.J);
      const Column c = column(a, g, j, lane, sfree[wave]);
      if (lane < a.W) {
        a.out_table[((size_t)g * a.W + lane) * a.J + j] = c.to;
        if (j == 0) a.out_lens[(size_t)g * a.W + lane] = c.len;
      }
    }
    return;
  }
  // A beam's copies in one pool.  Every wavefront works out the column.
  const PoolDesc& p = a.pool[blockIdx.y];
  for (int i = blockIdx.x; i < beams; i += gridDim.x) {
    const int g = i / a.W, w = i - g * a.W;
    const int par = min(max(a.parents[i], 0), a.W - 1);
    const int len = a.lens[(size_t)g * a.W + par];
    if (len <= 0) continue;
    const int j = len >> a.page_shift;
    if (j >= a.J || (len & (a.page - 1)) == 0) continue;  // no page that is in use
    const Column c = column(a, g, j, lane, sfree[wave]);
    if (!(__ballot(c.copies) >> w & 1)) continue;
    const int from = __shfl(c.from, w, 64), to = __shfl(c.to, w, 64), rows = __shfl(c.rows, w, 64);
    if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages) continue;
    const int bytes = (int)(((long long)rows * p.entries + a.page - 1) / a.page) * p.entry_bytes;  // of each head
    const char* const src = p.p + (size_t)from * p.page_stride;
    char* const dst = p.p + (size_t)to * p.page_stride;
    if (p.wide) {
      const int n = bytes / 16;
      for (int t = tid; t < n * p.heads; t += kReorderThreads) {
        const int h = t / n, o = t - h * n;
        const size_t at = (size_t)h * p.head_stride + (size_t)o * 16;
        *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
      }
    } else {
      const int n = bytes / 4;
      for (int t = tid; t < n * p.heads; t += kReorderThreads) {
        const int h = t / n, o = t - h * n;
        const size_t at = (size_t)h * p.head_stride + (size_t)o * 4;
        *reinterpret_cast<unsigned*>(dst + at) = *reinterpret_cast<const unsigned*>(src + at);
      }
    }
  }
}

}  // namespace

template <typename T>
hipError_t launch_select(const SelectArgs& a, hipStream_t stream) {
  const long long rows = (long long)a.B * a.W;
  const unsigned y = static_cast<unsigned>(std::min<long long>(rows, 32768));
  const dim3 grid(static_cast<unsigned>(a.segments), y, static_cast<unsigned>((rows + y - 1) / y));
  switch (a.per_segment / kSelectThreads) {
    case 4: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 4>), grid, dim3(kSelectThreads), 0, stream, a); break;
    case 8: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 8>), grid, dim3(kSelectThreads), 0, stream, a); break;
    case 16: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 16>), grid, dim3(kSelectThreads), 0, stream, a); break;
    default: hipLaunchKernelGGL((coalibi_select_rows_kernel<T, 32>), grid, dim3(kSelectThreads), 0, stream, a); break;
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
