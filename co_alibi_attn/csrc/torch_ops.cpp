// PyTorch-ROCm operators over the C ABI of libco_alibi (include/co_alibi.h).
//
//   co_alibi::fwd(q, k, v, slopes, causal, sm_scale, with_stats) -> (o, lse, stats)
//   co_alibi::bwd(do, q, k, v, o, lse, stats, slopes, causal, sm_scale) -> (dq, dk, dv)
//   co_alibi::bwd_dq(do, q, k, v, o, lse, stats, slopes, causal, sm_scale) -> dq
//   co_alibi::fwd_qkv(qkv, slopes, causal, sm_scale, with_stats) -> (o, lse, stats)
//   co_alibi::bwd_qkv(do, qkv, o, lse, stats, slopes, causal, sm_scale) -> dqkv
//   co_alibi::decode(q, k_cache, v_cache, slopes, seq_lens, max_seq_len, sm_scale, with_lse) -> (o, lse)
//   co_alibi::decode_tree(q, k, v, k_cache, v_cache, slopes, seq_lens, parents, block_table, max_seq_len, sm_scale,
//                         with_lse) -> (o, lse)
//   co_alibi::cache_append(k, v, k_cache!, v_cache!, seq_lens, counts, rows, block_table) -> ()
//   co_alibi::sample(logits, uniforms, temperature, top_k, top_p, min_p, their four values for every row) -> tokens
//   co_alibi::decode_tree_8bit(q, k, v, k_cache, v_cache, k_scale, v_scale, slopes, seq_lens, parents, block_table, max_seq_len,
//                              sm_scale, with_lse) -> (o, lse)
//   co_alibi::cache_append_8bit(k, v, k_cache!, v_cache!, k_scale!, v_scale!, seq_lens, counts, rows, block_table) -> ()
//   co_alibi::cache_read_8bit(k_cache, v_cache, k_scale, v_scale, seq_lens, first, block_table, rows, dtype) -> (k, v)
//   co_alibi::beam_select(logits, scores, finished, num_beams, end_token) -> (scores, parents, tokens)
//   co_alibi::cache_reorder(caches!, block_table, pages, seq_lens, parents, page_size) -> (block_table, seq_lens)
//
// They replace the reference's two Triton launches with their buffer set-up
// (co_alibi_attn/co_alibi_attn.py:35-57 and :83-133); decode and the operators after it have no counterpart there.  Each
// kernel runs on the caller's current HIP stream under a device guard of the inputs' device and
// allocates only through torch's caching allocator, so the operators can be captured in a HIP
// graph.  co_alibi::fwd carries its backward as a C++ autograd kernel: dQ alone runs backward
// pass 1 only (co_alibi::bwd_dq); any key / value gradient runs both passes (co_alibi::bwd).
// co_alibi::bwd uses the score store (pass 1 keeps s and dS, pass 2 reduces them) where the
// library has it and its workspace fits: at most CO_ALIBI_SCORE_STORE_LIMIT_MB megabytes (an
// environment variable read once; 16384 by default, 0 turns the store off) and at most half
// of the device memory that is free or cached by torch's allocator at the call.  If allocating
// it fails anyway, the backward takes the recompute path, whose workspace is O(S^2 / 32).
// The shape functions for FakeTensor / meta tracing are registered from Python.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cstdint>
#include <cstdlib>
#include <tuple>
#include <vector>

#include "../../include/co_alibi.h"

namespace {

using at::Tensor;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return CO_ALIBI_F32;
    case at::kHalf: return CO_ALIBI_F16;
    case at::kBFloat16: return CO_ALIBI_BF16;
    default: TORCH_CHECK_TYPE(false, "co_alibi: q, k, v must be float32, float16 or bfloat16, got ", t);
  }
  return -1;
}

void check(int rc) {
  TORCH_CHECK(rc == CO_ALIBI_OK, "co_alibi_attn: ", co_alibi_last_error(), " (status ", rc, ")");
}

// Contiguous tensor whose data pointer is 16-byte aligned (what the kernels load).
Tensor aligned(const Tensor& t) {
  Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}

// Whether the kernels can read a (B, H, S, D) operand in place (co_alibi_fwd_strided's rules), and its
// batch, head and row strides: those of dimensions of size 1 do not matter and are given as if
// contiguous, which the kernels have faster instantiations for.
struct Strides {
  long long v[3];
};
Strides strides_of(const Tensor& t) {
  const int64_t H = t.size(1), S = t.size(2), D = t.size(3);
  return {{t.size(0) == 1 ? H * S * D : t.stride(0), H == 1 ? S * D : t.stride(1), S == 1 ? D : t.stride(2)}};
}
bool readable(const Tensor& t) {
  const int64_t per16 = 16 / t.element_size();
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  const Strides s = strides_of(t);
  return s.v[0] % per16 == 0 && s.v[1] % per16 == 0 && s.v[2] % per16 == 0 && s.v[2] >= t.size(3) && s.v[2] <= 1 << 20;
}
// The operand itself where the kernels can read it in place, else a contiguous aligned copy.
Tensor in_place(const Tensor& t) { return readable(t) ? t : aligned(t); }
// An output itself where the kernels can write it in place, else a contiguous tensor to copy from (a
// packed projection's rows can be further apart than the kernels' 2^20 elements).
Tensor writable(const Tensor& t) { return readable(t) ? t : at::empty(t.sizes(), t.options()); }
// K and V, whose row strides must agree.
std::pair<Tensor, Tensor> kv_in_place(const Tensor& k, const Tensor& v) {
  if (readable(k) && readable(v) && strides_of(k).v[2] == strides_of(v).v[2]) return {k, v};
  return {aligned(k), aligned(v)};
}
template <size_t N>
std::array<long long, 3 * N> all_strides(const std::array<Tensor, N>& ts) {
  std::array<long long, 3 * N> out{};
  for (size_t i = 0; i < N; ++i) {
    const Strides s = strides_of(ts[i]);
    std::copy(s.v, s.v + 3, out.begin() + 3 * i);
  }
  return out;
}

// fp32 copy of the penalty slopes on the inputs' device (no copy when already so).
Tensor slopes_f32(const Tensor& slopes, const Tensor& like) {
  // (As the package hands them over: a detach alone costs the host half a microsecond a call.)
  if (slopes.scalar_type() == at::kFloat && slopes.device() == like.device() && slopes.is_contiguous()) return slopes;
  return slopes.detach().to(like.device(), at::kFloat).contiguous();
}

Tensor empty_stats(const Tensor& q) { return at::empty({0}, q.options().dtype(at::kFloat)); }

int64_t stats_numel(int64_t batch, int64_t heads_q, int64_t seq_q, int64_t seq_kv) {
  return static_cast<int64_t>(co_alibi_stats_numel(static_cast<int>(batch), static_cast<int>(heads_q),
                                                   static_cast<int>(seq_q), static_cast<int>(seq_kv)));
}

hipStream_t current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// ---------------------------------------------------------------------------- forward

// The forward into o (B, Hq, Sq, D); returns lse and stats (empty for inference).
std::tuple<Tensor, Tensor> launch_fwd(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& slopes,
                                      const Tensor& o, bool causal, double sm_scale, bool with_stats) {
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), seq_q = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1), seq_kv = k_in.size(2);
  c10::hip::HIPGuard guard(q_in.device().index());
  const Tensor q = in_place(q_in);
  const auto [k, v] = kv_in_place(k_in, v_in);
  const Tensor sl = slopes_f32(slopes, q);
  const auto f32 = q.options().dtype(at::kFloat);
  Tensor lse = with_stats ? at::empty({batch, heads_q, seq_q}, f32) : empty_stats(q);
  Tensor stats = with_stats ? at::empty({stats_numel(batch, heads_q, seq_q, seq_kv)}, f32) : empty_stats(q);
  // Inference: the tail skip with only its key-norm and work-order scratch.
  const size_t ws_bytes = with_stats ? 0 : co_alibi_fwd_inference_workspace_bytes(batch, heads_q, seq_q, seq_kv);
  Tensor ws;
  if (!with_stats) ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  const Tensor out = writable(o);
  const auto strides = all_strides<4>({q, k, v, out});
  check(co_alibi_fwd_strided(dtype_code(q.scalar_type()), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                             sl.data_ptr<float>(), out.data_ptr(), strides.data(),
                             with_stats ? lse.data_ptr<float>() : nullptr,
                             with_stats ? stats.data_ptr<float>() : nullptr, with_stats ? nullptr : ws.data_ptr(),
                             ws_bytes, batch, heads_q, heads_kv, seq_q, seq_kv, head_dim, causal ? 1 : 0,
                             static_cast<float>(sm_scale), current_stream(q)));
  if (!out.is_same(o)) o.copy_(out);
  return {lse, stats};
}

std::tuple<Tensor, Tensor, Tensor> fwd_hip(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                           const Tensor& slopes, bool causal, double sm_scale, bool with_stats) {
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), seq_q = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1), seq_kv = k_in.size(2);
  if (q_in.numel() == 0 || seq_kv == 0) {
    // Nothing to launch.  Rows that see no key get what the reference's l = 0 gives:
    // O = 0 / (0 + 1e-9) = 0 and LSE = -inf + log(1e-9) = -inf (co_alibi_fwd_kernel.py:115,120).
    Tensor o = at::zeros(q_in.sizes(), q_in.options());
    if (!with_stats) return {o, empty_stats(q_in), empty_stats(q_in)};
    Tensor lse = at::full({batch, heads_q, seq_q}, -std::numeric_limits<float>::infinity(),
                          q_in.options().dtype(at::kFloat));
    return {o, lse, at::zeros({stats_numel(batch, heads_q, seq_q, seq_kv)}, q_in.options().dtype(at::kFloat))};
  }
  Tensor o = at::empty(q_in.sizes(), q_in.options());
  auto [lse, stats] = launch_fwd(q_in, k_in, v_in, slopes, o, causal, sm_scale, with_stats);
  return {o, lse, stats};
}

// --------------------------------------------------------------------------- backward

// Largest workspace co_alibi::bwd takes for the score store (the environment's limit).
size_t score_store_limit() {
  static const size_t limit = [] {
    const char* e = std::getenv("CO_ALIBI_SCORE_STORE_LIMIT_MB");
    const long long mb = e != nullptr && *e != '\0' ? std::atoll(e) : 16384;
    return mb > 0 ? static_cast<size_t>(mb) << 20 : size_t{0};
  }();
  return limit;
}

// Device memory a new allocation can take on the current device: what the driver reports free
// plus what torch's caching allocator holds unused.
size_t device_memory_available() {
  size_t free_b = 0, total_b = 0;
  if (hipMemGetInfo(&free_b, &total_b) != hipSuccess) return 0;
  const auto stats = c10::hip::HIPCachingAllocator::getDeviceStats(c10::hip::current_device());
  const size_t agg = static_cast<size_t>(c10::CachingAllocator::StatType::AGGREGATE);
  const int64_t cached = stats.reserved_bytes[agg].current - stats.allocated_bytes[agg].current;
  return free_b + static_cast<size_t>(cached > 0 ? cached : 0);
}

// Shared set-up of the backward operators; stages 1 = pass 1 only (dq), 3 = both passes, into the
// given outputs (dk and dv undefined with stages 1).  The score-store path reads and writes every
// operand in place; the recompute path takes contiguous ones.
void launch_bwd(int stages, const Tensor& do_in, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                const Tensor& o_in, const Tensor& lse_in, const Tensor& stats_in, const Tensor& slopes, bool causal,
                double sm_scale, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), seq_q = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1), seq_kv = k_in.size(2);
  c10::hip::HIPGuard guard(q_in.device().index());
  const Tensor lse = lse_in.contiguous(), stats = stats_in.contiguous();
  const Tensor sl = slopes_f32(slopes, q_in);
  const int code = dtype_code(q_in.scalar_type());
  const int causal_i = causal ? 1 : 0;
  const float scale = static_cast<float>(sm_scale);
  const hipStream_t st = current_stream(q_in);
  const Tensor do_t = do_in.to(q_in.scalar_type());
  const auto bytes = q_in.options().dtype(at::kByte);
  if (stages & 2) {
    const size_t store_bytes =
        co_alibi_bwd_score_store_workspace_bytes(code, batch, heads_q, heads_kv, seq_q, seq_kv, head_dim, causal_i);
    Tensor ws;
    if (store_bytes != 0 && store_bytes <= score_store_limit() && store_bytes <= device_memory_available() / 2) {
      try {
        ws = at::empty({static_cast<int64_t>(store_bytes)}, bytes);
      } catch (const c10::OutOfMemoryError&) {  // the recompute path's smaller workspace below
      }
    }
    if (ws.defined()) {
      const Tensor q = in_place(q_in), o = in_place(o_in), dout = in_place(do_t);
      const auto [k, v] = kv_in_place(k_in, v_in);
      const std::array<Tensor, 3> to = {dq, dk, dv}, out = {writable(dq), writable(dk), writable(dv)};
      const auto strides = all_strides<8>({dout, q, k, v, o, out[0], out[1], out[2]});
      check(co_alibi_bwd_strided(code, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                 lse.data_ptr<float>(), stats.data_ptr<float>(), sl.data_ptr<float>(),
                                 out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), strides.data(),
                                 ws.data_ptr(), store_bytes, batch, heads_q, heads_kv, seq_q, seq_kv, head_dim,
                                 causal_i, scale, st));
      for (int i = 0; i < 3; ++i)
        if (!out[i].is_same(to[i])) to[i].copy_(out[i]);
      return;
    }
  }
  const Tensor q = aligned(q_in), k = aligned(k_in), v = aligned(v_in), o = aligned(o_in), dout = aligned(do_t);
  const size_t ws_bytes = co_alibi_bwd_workspace_bytes(batch, heads_q, seq_q, seq_kv);
  const Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, bytes);
  auto dense = [](const Tensor& t) { return t.defined() && !t.is_contiguous() ? at::empty(t.sizes(), t.options()) : t; };
  const Tensor cq = dense(dq), ck = dense(dk), cv = dense(dv);
  if (stages & 2) {
    check(co_alibi_bwd(code, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                       lse.data_ptr<float>(), stats.data_ptr<float>(), sl.data_ptr<float>(), cq.data_ptr(),
                       ck.data_ptr(), cv.data_ptr(), ws.data_ptr(), ws_bytes, batch, heads_q, heads_kv, seq_q, seq_kv,
                       head_dim, causal_i, scale, st));
  } else {
    check(co_alibi_bwd_dq(code, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                          lse.data_ptr<float>(), stats.data_ptr<float>(), sl.data_ptr<float>(), cq.data_ptr(),
                          ws.data_ptr(), ws_bytes, batch, heads_q, heads_kv, seq_q, seq_kv, head_dim, causal_i, scale,
                          st));
  }
  for (const auto& [to, from] : {std::pair(dq, cq), std::pair(dk, ck), std::pair(dv, cv)})
    if (to.defined() && !to.is_same(from)) to.copy_(from);
}

std::tuple<Tensor, Tensor, Tensor> bwd_common(int stages, const Tensor& dout, const Tensor& q, const Tensor& k,
                                              const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& stats,
                                              const Tensor& slopes, bool causal, double sm_scale) {
  if (q.numel() == 0 || k.numel() == 0) {  // no (query, key) pair: every gradient is zero
    return {at::zeros(q.sizes(), q.options()), at::zeros(k.sizes(), k.options()), at::zeros(v.sizes(), v.options())};
  }
  Tensor dq = at::empty(q.sizes(), q.options()), dk, dv;
  if (stages & 2) {
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  launch_bwd(stages, dout, q, k, v, o, lse, stats, slopes, causal, sm_scale, dq, dk, dv);
  return {dq, dk, dv};
}

std::tuple<Tensor, Tensor, Tensor> bwd_hip(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                                           const Tensor& o, const Tensor& lse, const Tensor& stats,
                                           const Tensor& slopes, bool causal, double sm_scale) {
  return bwd_common(3, dout, q, k, v, o, lse, stats, slopes, causal, sm_scale);
}

Tensor bwd_dq_hip(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                  const Tensor& lse, const Tensor& stats, const Tensor& slopes, bool causal, double sm_scale) {
  return std::get<0>(bwd_common(1, dout, q, k, v, o, lse, stats, slopes, causal, sm_scale));
}

// ------------------------------------------------------------------------- packed QKV

// Part i (0 q, 1 k, 2 v) of a packed (B, S, 3, H, D) tensor, and any (B, S, H, D) tensor, as (B, H, S, D).
Tensor qkv_part(const Tensor& qkv, int64_t i) { return qkv.select(2, i).transpose(1, 2); }

// Attention of a fused projection's output, read in place; o is (B, S, H, D) contiguous, which the
// output projection reads without a copy.
std::tuple<Tensor, Tensor, Tensor> fwd_qkv_hip(const Tensor& qkv, const Tensor& slopes, bool causal, double sm_scale,
                                               bool with_stats) {
  const Tensor q = qkv_part(qkv, 0), k = qkv_part(qkv, 1), v = qkv_part(qkv, 2);
  const std::vector<int64_t> shape{qkv.size(0), qkv.size(1), qkv.size(3), qkv.size(4)};
  if (qkv.numel() == 0) {
    Tensor o, lse, stats;
    std::tie(o, lse, stats) = fwd_hip(q, k, v, slopes, causal, sm_scale, with_stats);
    return {at::zeros(shape, qkv.options()), lse, stats};
  }
  Tensor o = at::empty(shape, qkv.options());
  auto [lse, stats] = launch_fwd(q, k, v, slopes, o.transpose(1, 2), causal, sm_scale, with_stats);
  return {o, lse, stats};
}

// Its gradient, written into one packed tensor (no per-part gradients to zero-fill and add up).
Tensor bwd_qkv_hip(const Tensor& dout, const Tensor& qkv, const Tensor& o, const Tensor& lse, const Tensor& stats,
                   const Tensor& slopes, bool causal, double sm_scale) {
  if (qkv.numel() == 0) return at::zeros(qkv.sizes(), qkv.options());
  Tensor dqkv = at::empty(qkv.sizes(), qkv.options());
  launch_bwd(3, dout.transpose(1, 2), qkv_part(qkv, 0), qkv_part(qkv, 1), qkv_part(qkv, 2), o.transpose(1, 2), lse,
             stats, slopes, causal, sm_scale, qkv_part(dqkv, 0), qkv_part(dqkv, 1), qkv_part(dqkv, 2));
  return dqkv;
}

// ----------------------------------------------------------------------------- decode

std::tuple<Tensor, Tensor> decode_hip(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& slopes,
                                      const c10::optional<Tensor>& seq_lens, int64_t max_seq_len, double sm_scale,
                                      bool with_lse) {
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1), capacity = k_in.size(2);
  if (q_in.numel() == 0) {  // an empty batch
    Tensor o = at::empty(q_in.sizes(), q_in.options());
    Tensor lse = with_lse ? at::empty({batch, heads_q, 1}, q_in.options().dtype(at::kFloat)) : empty_stats(q_in);
    return {o, lse};
  }
  c10::hip::HIPGuard guard(q_in.device().index());
  if (head_dim == 16) {
    // The decode kernels have no head dim of 16: run on heads padded to 32 with zero columns
    // (the products over d are unchanged, the padding columns of O come out zero) and return
    // the first 16 columns.  This copies the caches once per step.
    auto [o32, lse] = decode_hip(at::constant_pad_nd(q_in, {0, 16}), at::constant_pad_nd(k_in, {0, 16}),
                                 at::constant_pad_nd(v_in, {0, 16}), slopes, seq_lens, max_seq_len, sm_scale, with_lse);
    return {o32.narrow(3, 0, 16).contiguous(), lse};
  }
  const Tensor q = aligned(q_in), k = aligned(k_in), v = aligned(v_in);
  Tensor lens;
  if (seq_lens.has_value() && seq_lens->defined()) lens = seq_lens->to(q.device(), at::kInt).contiguous();
  const Tensor sl = slopes_f32(slopes, q);
  Tensor o = at::empty_like(q);
  Tensor lse = with_lse ? at::empty({batch, heads_q, 1}, q.options().dtype(at::kFloat)) : empty_stats(q);
  const size_t ws_bytes = co_alibi_decode_workspace_bytes(batch, heads_q, max_seq_len, head_dim);
  Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  check(co_alibi_decode(dtype_code(q.scalar_type()), q.data_ptr(), k.data_ptr(), v.data_ptr(), sl.data_ptr<float>(),
                        lens.defined() ? lens.data_ptr<int>() : nullptr, o.data_ptr(),
                        with_lse ? lse.data_ptr<float>() : nullptr, ws.data_ptr(), ws_bytes, batch, heads_q, heads_kv,
                        max_seq_len, capacity, head_dim, static_cast<float>(sm_scale), current_stream(q)));
  return {o, lse};
}

// ----------------------------------------------------------------------- serving step

// An index array as the kernels read it (int32, dense, on `like`'s device); 64-bit values that do not fit are
// clamped, not wrapped into the valid range.
Tensor index_i32(const Tensor& t, const Tensor& like) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong,
                   "co_alibi: lengths, tables and indices must be int32 or int64, got ", t.scalar_type());
  const Tensor d = t.to(like.device());
  if (d.scalar_type() == at::kInt) return d.contiguous();
  return d.clamp(std::numeric_limits<int>::min(), std::numeric_limits<int>::max()).to(at::kInt).contiguous();
}
const int* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr<int>() : nullptr; }
bool given(const c10::optional<Tensor>& t) { return t.has_value() && t->defined(); }

// The caches of a call over `batch` sequences: pools of pages with a table, else one cache per sequence.  They
// are read and written in place, never copied, so a layout the kernels cannot address is refused.
struct Caches {
  Tensor table;  // int32 (batch, blocks), or undefined
  int64_t blocks = 0, units = 0, page = 0, capacity = 0;
};
Caches check_caches(const char* fn, const Tensor& like, int64_t batch, const Tensor& k_cache, const Tensor& v_cache,
                    const c10::optional<Tensor>& block_table, bool eight = false) {
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(), fn,
                    ": k_cache and v_cache must be 4-dimensional and of one shape, got ", k_cache.sizes(), " and ",
                    v_cache.sizes());
  TORCH_CHECK_TYPE(eight || (k_cache.scalar_type() == like.scalar_type() && v_cache.scalar_type() == like.scalar_type()), fn,
                   ": the caches' dtype must be the new tokens', ", like.scalar_type(), ", got ", k_cache.scalar_type(),
                   " and ", v_cache.scalar_type());
  TORCH_CHECK_VALUE(k_cache.device() == like.device() && v_cache.device() == like.device(), fn,
                    ": the caches must be on the new tokens' device");
  Caches c;
  c.units = k_cache.size(0);
  c.page = k_cache.size(2);
  if (given(block_table)) {
    TORCH_CHECK_VALUE(block_table->dim() == 2 && block_table->size(0) == batch, fn, ": block_table must be (", batch,
                      ", blocks), got ", block_table->sizes());
    c.table = index_i32(*block_table, like);
    c.blocks = c.table.size(1);
    TORCH_CHECK_VALUE(c.page >= 16 && (c.page & (c.page - 1)) == 0, fn, ": a page must hold a power of two >= 16 rows, got ",
                      c.page);
    c.capacity = c.blocks * c.page;
  } else {
    TORCH_CHECK_VALUE(c.units == batch, fn, ": without a block_table the caches hold one entry per sequence, got ", c.units,
                      " for ", batch);
    c.capacity = c.page;
  }
  TORCH_CHECK_VALUE(c.capacity <= 1 << 30, fn, ": a sequence's cache holds at most 2^30 rows");
  if (k_cache.numel() != 0)
    TORCH_CHECK_VALUE(readable(k_cache) && readable(v_cache), fn,
                      ": a cache's rows must be dense, 16-byte aligned and at most 2^20 elements apart");
  return c;
}
int as_int(const char* fn, const char* name, int64_t x) {
  TORCH_CHECK_VALUE(x >= 0 && x <= std::numeric_limits<int>::max(), fn, ": ", name, " out of range: ", x);
  return static_cast<int>(x);
}

// What the tree decodes check of their inputs, and the index arrays as the kernels read them.
struct TreeInputs {
  int code;
  Caches caches;
  Tensor lens, parents;
};
TreeInputs check_tree(const char* fn, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache,
                      const Tensor& v_cache, const Tensor& slopes, const c10::optional<Tensor>& seq_lens,
                      const c10::optional<Tensor>& parents, const c10::optional<Tensor>& block_table, int64_t max_seq_len,
                      bool eight) {
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && v_in.sizes() == k_in.sizes(), fn,
                    ": q must be (B, Hq, T, D) and k, v (B, Hkv, T, D), got ", q_in.sizes(), ", ", k_in.sizes(), " and ",
                    v_in.sizes());
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), tokens = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1);
  TORCH_CHECK_VALUE(k_in.size(0) == batch && k_in.size(2) == tokens && k_in.size(3) == head_dim, fn,
                    ": k and v must hold q's batch, tokens and head dim, got ", k_in.sizes(), " for ", q_in.sizes());
  TORCH_CHECK_TYPE(k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type(), fn,
                   ": q, k and v must share one dtype");
  TORCH_CHECK_VALUE(k_in.device() == q_in.device() && v_in.device() == q_in.device(), fn,
                    ": q, k and v must be on one device");
  TreeInputs in;
  in.code = dtype_code(q_in.scalar_type());
  c10::hip::HIPGuard guard(q_in.device().index());
  in.caches = check_caches(fn, q_in, batch, k_cache, v_cache, block_table, eight);
  const Caches& c = in.caches;
  TORCH_CHECK_VALUE(k_cache.size(1) == heads_kv && k_cache.size(3) == head_dim, fn,
                    ": the caches must have k's heads and head dim, got ", k_cache.sizes(), " for ", k_in.sizes());
  TORCH_CHECK_VALUE(slopes.dim() == 1 && slopes.size(0) == heads_q, fn, ": slopes must be (", heads_q, ",), got ", slopes.sizes());
  TORCH_CHECK_VALUE(max_seq_len >= 0 && max_seq_len <= c.capacity, fn, ": max_seq_len must be in [0, ", c.capacity, "], got ",
                    max_seq_len);
  if (given(seq_lens)) {
    TORCH_CHECK_VALUE(seq_lens->dim() == 1 && seq_lens->size(0) == batch, fn, ": seq_lens must be (", batch, ",), got ",
                      seq_lens->sizes());
    in.lens = index_i32(*seq_lens, q_in);
  }
  if (given(parents)) {
    const bool one = parents->dim() == 1 && parents->size(0) == tokens;
    TORCH_CHECK_VALUE(one || (parents->dim() == 2 && parents->size(0) == batch && parents->size(1) == tokens), fn,
                      ": parents must be (", tokens, ",) or (", batch, ", ", tokens, "), got ", parents->sizes());
    in.parents = index_i32(*parents, q_in);
  }
  return in;
}

std::tuple<Tensor, Tensor> decode_tree_hip(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                           const Tensor& k_cache, const Tensor& v_cache, const Tensor& slopes,
                                           const c10::optional<Tensor>& seq_lens, const c10::optional<Tensor>& parents,
                                           const c10::optional<Tensor>& block_table, int64_t max_seq_len, double sm_scale,
                                           bool with_lse) {
  const char* fn = "co_alibi::decode_tree";
  const auto [code, c, lens, par] =
      check_tree(fn, q_in, k_in, v_in, k_cache, v_cache, slopes, seq_lens, parents, block_table, max_seq_len, false);
  c10::hip::HIPGuard guard(q_in.device().index());
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), tokens = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1);
  const auto f32 = q_in.options().dtype(at::kFloat);
  Tensor o = at::empty(q_in.sizes(), q_in.options());
  Tensor lse = with_lse ? at::empty({batch, heads_q, tokens}, f32) : empty_stats(q_in);
  if (q_in.numel() == 0) return {o, lse};
  const Tensor q = in_place(q_in), k = in_place(k_in), v = in_place(v_in);
  // A pool without rows, or behind a table without blocks, is never read; the launch wants an address all the same.
  const bool none = k_cache.numel() == 0 || c.capacity == 0;
  const Tensor kc = none ? k : k_cache, vc = none ? v : v_cache;
  TORCH_CHECK_VALUE(!none || max_seq_len == 0, fn, ": the caches hold no rows");
  const Tensor sl = slopes_f32(slopes, q);
  const size_t ws_bytes = co_alibi_decode_tree_workspace_bytes(code, as_int(fn, "batch", batch), as_int(fn, "heads", heads_q),
                                                               as_int(fn, "heads", heads_kv), as_int(fn, "tokens", tokens),
                                                               as_int(fn, "max_seq_len", max_seq_len),
                                                               as_int(fn, "head_dim", head_dim));
  Tensor ws;
  if (ws_bytes != 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  const auto strides = all_strides<5>({q, k, v, kc, vc});
  check(co_alibi_decode_tree(code, q.data_ptr(), k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), strides.data(),
                             sl.data_ptr<float>(), data_or_null(lens), data_or_null(par),
                             par.defined() && par.dim() == 2 ? 1 : 0, none ? nullptr : data_or_null(c.table),
                             as_int(fn, "blocks", c.blocks), as_int(fn, "pages", c.units),
                             none ? 1 : as_int(fn, "page", c.page), o.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr,
                             ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, batch, heads_q, heads_kv, tokens, max_seq_len,
                             head_dim, static_cast<float>(sm_scale), current_stream(q)));
  return {o, lse};
}

// What the appends check of their inputs, and the index arrays as the kernels read them.
struct AppendInputs {
  int code;
  Caches caches;
  Tensor lens, counts, rows;
  int64_t new_rows;
};
AppendInputs check_append(const char* fn, const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                          const Tensor& seq_lens, const c10::optional<Tensor>& counts, const c10::optional<Tensor>& rows,
                          const c10::optional<Tensor>& block_table, bool eight) {
  TORCH_CHECK_VALUE(k_in.dim() == 4 && v_in.sizes() == k_in.sizes(), fn, ": k and v must be (B, Hkv, T, D), got ",
                    k_in.sizes(), " and ", v_in.sizes());
  TORCH_CHECK_TYPE(v_in.scalar_type() == k_in.scalar_type(), fn, ": k and v must share one dtype");
  TORCH_CHECK_VALUE(v_in.device() == k_in.device(), fn, ": k and v must be on one device");
  const int64_t batch = k_in.size(0), heads_kv = k_in.size(1), tokens = k_in.size(2), head_dim = k_in.size(3);
  AppendInputs in;
  in.code = dtype_code(k_in.scalar_type());
  c10::hip::HIPGuard guard(k_in.device().index());
  in.caches = check_caches(fn, k_in, batch, k_cache, v_cache, block_table, eight);
  TORCH_CHECK_VALUE(k_cache.size(1) == heads_kv && k_cache.size(3) == head_dim, fn,
                    ": the caches must have k's heads and head dim, got ", k_cache.sizes(), " for ", k_in.sizes());
  TORCH_CHECK_VALUE(seq_lens.dim() == 1 && seq_lens.size(0) == batch, fn, ": seq_lens must be (", batch, ",), got ",
                    seq_lens.sizes());
  in.lens = index_i32(seq_lens, k_in);
  if (given(counts)) {
    TORCH_CHECK_VALUE(counts->dim() == 1 && counts->size(0) == batch, fn, ": counts must be (", batch, ",), got ",
                      counts->sizes());
    in.counts = index_i32(*counts, k_in);
  }
  in.new_rows = tokens;
  if (given(rows)) {
    TORCH_CHECK_VALUE(rows->dim() == 2 && rows->size(0) == batch, fn, ": rows must be (", batch, ", n), got ", rows->sizes());
    in.rows = index_i32(*rows, k_in);
    in.new_rows = in.rows.size(1);
  }
  return in;
}

void cache_append_hip(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                      const Tensor& seq_lens, const c10::optional<Tensor>& counts, const c10::optional<Tensor>& rows,
                      const c10::optional<Tensor>& block_table) {
  const char* fn = "co_alibi::cache_append";
  const auto [code, c, lens, cnt, idx, new_rows] =
      check_append(fn, k_in, v_in, k_cache, v_cache, seq_lens, counts, rows, block_table, false);
  c10::hip::HIPGuard guard(k_in.device().index());
  const int64_t batch = k_in.size(0), heads_kv = k_in.size(1), tokens = k_in.size(2), head_dim = k_in.size(3);
  if (k_in.numel() == 0 || new_rows == 0 || k_cache.numel() == 0 || c.capacity == 0) return;
  const Tensor k = in_place(k_in), v = in_place(v_in);
  const auto strides = all_strides<4>({k, v, k_cache, v_cache});
  check(co_alibi_cache_append(code, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), strides.data(),
                              lens.data_ptr<int>(), data_or_null(cnt), data_or_null(idx), as_int(fn, "rows", new_rows),
                              data_or_null(c.table), as_int(fn, "blocks", c.blocks), as_int(fn, "pages", c.units),
                              as_int(fn, "page", c.page), as_int(fn, "batch", batch), as_int(fn, "heads", heads_kv),
                              as_int(fn, "tokens", tokens), as_int(fn, "head_dim", head_dim), current_stream(k)));
  for (const Tensor* t : {&k_cache, &v_cache})  // autograd's record of a write in place
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// An 8-bit cache: its format, and the scales beside its codes, read and written in place, too.
int format_code(const char* fn, const Tensor& k_cache, const Tensor& v_cache) {
  const auto t = k_cache.scalar_type();
  TORCH_CHECK_TYPE((t == at::kFloat8_e4m3fn || t == at::kChar) && v_cache.scalar_type() == t, fn,
                   ": the caches must both be float8_e4m3fn or int8, got ", t, " and ", v_cache.scalar_type());
  return t == at::kChar ? CO_ALIBI_INT8 : CO_ALIBI_E4M3;
}
struct Scales {
  std::array<long long, 4> strides;  // (unit, head) of k's, then of v's
};
Scales check_scales(const char* fn, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale) {
  const std::array<int64_t, 3> want{k_cache.size(0), k_cache.size(1), (k_cache.size(2) + 15) / 16};
  for (const Tensor* t : {&k_scale, &v_scale}) {
    TORCH_CHECK_VALUE(t->sizes() == at::IntArrayRef(want), fn, ": the scales must be ", at::IntArrayRef(want), ", got ", t->sizes());
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, fn, ": the scales must be float32, got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->device() == k_cache.device(), fn, ": the scales must be on the caches' device");
    TORCH_CHECK_VALUE(t->size(2) <= 1 || t->stride(2) == 1, fn, ": a head's scales must follow one another");
  }
  for (const Tensor* t : {&k_cache, &v_cache})
    TORCH_CHECK_VALUE(t->numel() == 0 || t->size(2) == 1 || t->stride(2) == t->size(3), fn,
                      ": the rows of an 8-bit cache must be dense");
  return {{k_scale.stride(0), k_scale.stride(1), v_scale.stride(0), v_scale.stride(1)}};
}

std::tuple<Tensor, Tensor> decode_tree_8bit_hip(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                                const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                                                const Tensor& v_scale, const Tensor& slopes,
                                                const c10::optional<Tensor>& seq_lens, const c10::optional<Tensor>& parents,
                                                const c10::optional<Tensor>& block_table, int64_t max_seq_len,
                                                double sm_scale, bool with_lse) {
  const char* fn = "co_alibi::decode_tree_8bit";
  const TreeInputs in = check_tree(fn, q_in, k_in, v_in, k_cache, v_cache, slopes, seq_lens, parents, block_table, max_seq_len, true);
  const int format = format_code(fn, k_cache, v_cache);
  const Scales sc = check_scales(fn, k_cache, v_cache, k_scale, v_scale);
  c10::hip::HIPGuard guard(q_in.device().index());
  const int64_t batch = q_in.size(0), heads_q = q_in.size(1), tokens = q_in.size(2), head_dim = q_in.size(3);
  const int64_t heads_kv = k_in.size(1);
  Tensor o = at::empty(q_in.sizes(), q_in.options());
  Tensor lse = with_lse ? at::empty({batch, heads_q, tokens}, q_in.options().dtype(at::kFloat)) : empty_stats(q_in);
  if (q_in.numel() == 0) return {o, lse};
  const Tensor q = in_place(q_in), k = in_place(k_in), v = in_place(v_in);
  // A pool without rows, or behind a table without blocks, is never read; the launch wants addresses all the same.
  const bool none = k_cache.numel() == 0 || in.caches.capacity == 0;
  TORCH_CHECK_VALUE(!none || max_seq_len == 0, fn, ": the caches hold no rows");
  const Tensor sl = slopes_f32(slopes, q);
  const size_t ws_bytes = co_alibi_decode_tree_8bit_workspace_bytes(
      in.code, as_int(fn, "batch", batch), as_int(fn, "heads", heads_q), as_int(fn, "heads", heads_kv),
      as_int(fn, "tokens", tokens), as_int(fn, "max_seq_len", max_seq_len), as_int(fn, "head_dim", head_dim));
  Tensor ws;
  if (ws_bytes != 0) ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  const auto new_strides = all_strides<3>({q, k, v});
  std::array<long long, 15> strides{};
  std::copy(new_strides.begin(), new_strides.end(), strides.begin());
  strides[11] = strides[14] = head_dim;
  if (!none) {
    const auto cache_strides = all_strides<2>({k_cache, v_cache});
    std::copy(cache_strides.begin(), cache_strides.end(), strides.begin() + 9);
  }
  const void* const spare = k.data_ptr();
  check(co_alibi_decode_tree_8bit(
      in.code, format, q.data_ptr(), k.data_ptr(), v.data_ptr(), none ? spare : k_cache.data_ptr(),
      none ? spare : v_cache.data_ptr(), none ? static_cast<const float*>(spare) : k_scale.data_ptr<float>(),
      none ? static_cast<const float*>(spare) : v_scale.data_ptr<float>(), strides.data(), sc.strides.data(),
      sl.data_ptr<float>(), data_or_null(in.lens), data_or_null(in.parents),
      in.parents.defined() && in.parents.dim() == 2 ? 1 : 0, none ? nullptr : data_or_null(in.caches.table),
      as_int(fn, "blocks", in.caches.blocks), as_int(fn, "pages", in.caches.units),
      none ? 1 : as_int(fn, "page", in.caches.page), o.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr,
      ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, batch, heads_q, heads_kv, tokens, max_seq_len, head_dim,
      static_cast<float>(sm_scale), current_stream(q)));
  return {o, lse};
}

void cache_append_8bit_hip(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                           const Tensor& k_scale, const Tensor& v_scale, const Tensor& seq_lens,
                           const c10::optional<Tensor>& counts, const c10::optional<Tensor>& rows,
                           const c10::optional<Tensor>& block_table) {
  const char* fn = "co_alibi::cache_append_8bit";
  const AppendInputs in = check_append(fn, k_in, v_in, k_cache, v_cache, seq_lens, counts, rows, block_table, true);
  const int format = format_code(fn, k_cache, v_cache);
  const Scales sc = check_scales(fn, k_cache, v_cache, k_scale, v_scale);
  c10::hip::HIPGuard guard(k_in.device().index());
  if (k_in.numel() == 0 || in.new_rows == 0 || k_cache.numel() == 0 || in.caches.capacity == 0) return;
  const Tensor k = in_place(k_in), v = in_place(v_in);
  const auto strides = all_strides<4>({k, v, k_cache, v_cache});
  check(co_alibi_cache_append_8bit(in.code, format, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                   k_scale.data_ptr<float>(), v_scale.data_ptr<float>(), strides.data(), sc.strides.data(),
                                   in.lens.data_ptr<int>(), data_or_null(in.counts), data_or_null(in.rows),
                                   as_int(fn, "rows", in.new_rows), data_or_null(in.caches.table),
                                   as_int(fn, "blocks", in.caches.blocks), as_int(fn, "pages", in.caches.units),
                                   as_int(fn, "page", in.caches.page), as_int(fn, "batch", k_in.size(0)),
                                   as_int(fn, "heads", k_in.size(1)), as_int(fn, "tokens", k_in.size(2)),
                                   as_int(fn, "head_dim", k_in.size(3)), current_stream(k)));
  for (const Tensor* t : {&k_cache, &v_cache, &k_scale, &v_scale})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

std::tuple<Tensor, Tensor> cache_read_8bit_hip(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                                               const Tensor& v_scale, const Tensor& seq_lens,
                                               const c10::optional<Tensor>& first, const c10::optional<Tensor>& block_table,
                                               int64_t rows, at::ScalarType dtype) {
  const char* fn = "co_alibi::cache_read_8bit";
  TORCH_CHECK_VALUE(seq_lens.dim() == 1, fn, ": seq_lens must be (B,), got ", seq_lens.sizes());
  const int64_t batch = seq_lens.size(0);
  const int code = dtype_code(dtype), format = format_code(fn, k_cache, v_cache);
  c10::hip::HIPGuard guard(k_cache.device().index());
  const Caches c = check_caches(fn, k_cache, batch, k_cache, v_cache, block_table, true);
  const Scales sc = check_scales(fn, k_cache, v_cache, k_scale, v_scale);
  const Tensor lens = index_i32(seq_lens, k_cache);
  Tensor from;
  if (given(first)) {
    TORCH_CHECK_VALUE(first->dim() == 1 && first->size(0) == batch, fn, ": first must be (", batch, ",), got ", first->sizes());
    from = index_i32(*first, k_cache);
  }
  TORCH_CHECK_VALUE(rows >= 0, fn, ": rows must be >= 0, got ", rows);
  const int64_t heads = k_cache.size(1), head_dim = k_cache.size(3);
  const auto options = k_cache.options().dtype(dtype);
  if (k_cache.numel() == 0 || c.capacity == 0) {
    Tensor k = at::zeros({batch, heads, rows, head_dim}, options), v = at::zeros_like(k);
    if (k.numel() != 0 && c.capacity != 0) {  // a pool without pages: filled rows lie outside it
      Tensor row = at::arange(rows, lens.options().dtype(at::kLong)).unsqueeze(0);
      if (from.defined()) row = row + from.unsqueeze(1);
      const Tensor filled = row.ge(0).logical_and(row.lt(lens.clamp_max(c.capacity).unsqueeze(1)));
      for (const Tensor& t : {k, v}) t.masked_fill_(filled.unsqueeze(1).unsqueeze(3), std::numeric_limits<double>::quiet_NaN());
    }
    return {k, v};
  }
  Tensor k = at::empty({batch, heads, rows, head_dim}, options), v = at::empty_like(k);
  if (k.numel() == 0) return {k, v};
  const auto strides = all_strides<2>({k_cache, v_cache});
  check(co_alibi_cache_read_8bit(code, format, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr<float>(),
                                 v_scale.data_ptr<float>(), strides.data(), sc.strides.data(), lens.data_ptr<int>(),
                                 data_or_null(from), as_int(fn, "rows", rows), data_or_null(c.table),
                                 as_int(fn, "blocks", c.blocks), as_int(fn, "pages", c.units), as_int(fn, "page", c.page),
                                 k.data_ptr(), v.data_ptr(), as_int(fn, "batch", batch), as_int(fn, "heads", heads),
                                 as_int(fn, "head_dim", head_dim), current_stream(k_cache)));
  return {k, v};
}

std::tuple<Tensor, Tensor, Tensor> beam_select_hip(const Tensor& logits_in, const Tensor& scores_in,
                                                   const c10::optional<Tensor>& finished, int64_t num_beams,
                                                   int64_t end_token) {
  const char* fn = "co_alibi::beam_select";
  TORCH_CHECK_VALUE(logits_in.dim() == 3, fn, ": logits must be (B, W, V), got ", logits_in.sizes());
  const int64_t batch = logits_in.size(0), beams = logits_in.size(1), vocab = logits_in.size(2);
  const int code = dtype_code(logits_in.scalar_type());
  TORCH_CHECK_VALUE(scores_in.dim() == 2 && scores_in.size(0) == batch && scores_in.size(1) == beams, fn, ": scores must be (",
                    batch, ", ", beams, "), got ", scores_in.sizes());
  TORCH_CHECK_TYPE(scores_in.scalar_type() == at::kFloat, fn, ": scores must be float32, got ", scores_in.scalar_type());
  c10::hip::HIPGuard guard(logits_in.device().index());
  Tensor done;
  if (given(finished)) {
    TORCH_CHECK_VALUE(finished->sizes() == scores_in.sizes(), fn, ": finished must be (", batch, ", ", beams, "), got ",
                      finished->sizes());
    TORCH_CHECK_TYPE(finished->scalar_type() == at::kBool, fn, ": finished must be bool, got ", finished->scalar_type());
    done = finished->to(logits_in.device()).contiguous();
  }
  Tensor scores = at::empty({batch, num_beams}, logits_in.options().dtype(at::kFloat));
  Tensor parents = at::empty({batch, num_beams}, logits_in.options().dtype(at::kInt));
  Tensor tokens = at::empty({batch, num_beams}, logits_in.options().dtype(at::kLong));
  if (batch == 0) return {scores, parents, tokens};
  const Tensor logits = logits_in.stride(2) == 1 || vocab == 1 ? logits_in : logits_in.contiguous();
  const Tensor from = scores_in.to(logits.device()).contiguous();
  const size_t ws_bytes = co_alibi_beam_select_workspace_bytes(code, as_int(fn, "batch", batch), as_int(fn, "beams", beams),
                                                               as_int(fn, "num_beams", num_beams), as_int(fn, "vocab", vocab));
  Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, logits.options().dtype(at::kByte));
  const std::array<long long, 2> strides{batch == 1 ? beams * vocab : logits.stride(0), beams == 1 ? vocab : logits.stride(1)};
  check(co_alibi_beam_select(code, logits.data_ptr(), strides.data(), from.data_ptr<float>(),
                             done.defined() ? reinterpret_cast<const unsigned char*>(done.data_ptr<bool>()) : nullptr,
                             as_int(fn, "end_token", end_token), scores.data_ptr<float>(), parents.data_ptr<int>(),
                             reinterpret_cast<long long*>(tokens.data_ptr<int64_t>()), ws.data_ptr(), ws_bytes, batch, beams,
                             num_beams, vocab, current_stream(logits)));
  return {scores, parents, tokens};
}

std::tuple<Tensor, Tensor> cache_reorder_hip(at::TensorList caches, const Tensor& block_table, const Tensor& pages,
                                             const Tensor& seq_lens, const Tensor& parents, int64_t page_size) {
  const char* fn = "co_alibi::cache_reorder";
  TORCH_CHECK_VALUE(parents.dim() == 2, fn, ": parents must be (B, W), got ", parents.sizes());
  const int64_t batch = parents.size(0), beams = parents.size(1);
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.size(0) == batch * beams && pages.sizes() == block_table.sizes(), fn,
                    ": block_table and pages must be (", batch * beams, ", blocks), got ", block_table.sizes(), " and ",
                    pages.sizes());
  TORCH_CHECK_VALUE(seq_lens.dim() == 1 && seq_lens.size(0) == batch * beams, fn, ": seq_lens must be (", batch * beams,
                    ",), got ", seq_lens.sizes());
  TORCH_CHECK_VALUE(!caches.empty(), fn, ": there are no caches");
  const Tensor& like = caches[0];
  c10::hip::HIPGuard guard(like.device().index());
  std::vector<void*> pools;
  std::vector<long long> shapes;
  const int64_t num_pages = like.size(0);
  for (const Tensor& t : caches) {
    TORCH_CHECK_VALUE(t.dim() >= 3 && t.size(0) == num_pages, fn, ": the caches must be (", num_pages,
                      " pages, heads, rows of a page, ...), got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == like.device() && t.device().is_cuda(), fn, ": the caches must be on one CUDA device");
    TORCH_CHECK_VALUE(!t.requires_grad(), fn, ": the caches are written in place and cannot require gradients");
    int64_t entry = t.element_size();
    for (int64_t d = t.dim() - 1; d >= 3; --d) {
      TORCH_CHECK_VALUE(t.size(d) == 1 || t.stride(d) * t.element_size() == entry, fn, ": the rows of a page's head must be dense");
      entry *= t.size(d);
    }
    TORCH_CHECK_VALUE(t.size(2) == 1 || t.stride(2) * t.element_size() == entry, fn, ": the rows of a page's head must be dense");
    if (t.numel() == 0) continue;
    pools.push_back(t.data_ptr());
    for (long long x : {static_cast<long long>(t.stride(0) * t.element_size()), static_cast<long long>(t.stride(1) * t.element_size()),
                        static_cast<long long>(t.size(1)), static_cast<long long>(t.size(2)), static_cast<long long>(entry)})
      shapes.push_back(x);
  }
  const Tensor table = index_i32(block_table, like), home = index_i32(pages, like), lens = index_i32(seq_lens, like),
               par = index_i32(parents, like);
  Tensor out_table = at::empty(table.sizes(), table.options()), out_lens = at::empty(lens.sizes(), lens.options());
  if (table.numel() == 0) {
    TORCH_CHECK_VALUE(lens.numel() == 0, fn, ": the block table has no blocks");
    return {out_table, out_lens};
  }
  TORCH_CHECK_VALUE(!pools.empty(), fn, ": the caches are empty");
  check(co_alibi_cache_reorder(pools.data(), shapes.data(), static_cast<int>(pools.size()), table.data_ptr<int>(),
                               home.data_ptr<int>(), lens.data_ptr<int>(), par.data_ptr<int>(), out_table.data_ptr<int>(),
                               out_lens.data_ptr<int>(), as_int(fn, "batch", batch), as_int(fn, "beams", beams),
                               as_int(fn, "blocks", table.size(1)), as_int(fn, "pages", num_pages),
                               as_int(fn, "page_size", page_size), current_stream(like)));
  for (const Tensor& t : caches)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return {out_table, out_lens};
}

// A setting with one value per row, as the kernel reads it.
template <typename V>
const V* setting(const char* fn, const char* name, const c10::optional<Tensor>& t, const Tensor& logits, at::ScalarType type,
                 Tensor& keep) {
  if (!given(t)) return nullptr;
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == logits.size(0), fn, ": ", name, " must be one value or (", logits.size(0),
                    ",), got ", t->sizes());
  keep = type == at::kInt ? index_i32(*t, logits) : t->to(logits.device(), type).contiguous();
  return keep.data_ptr<V>();
}

Tensor sample_hip(const Tensor& logits_in, const Tensor& uniforms, const c10::optional<Tensor>& temperature,
                  const c10::optional<Tensor>& top_k, const c10::optional<Tensor>& top_p, const c10::optional<Tensor>& min_p,
                  double temperature_all, int64_t top_k_all, double top_p_all, double min_p_all) {
  const char* fn = "co_alibi::sample";
  TORCH_CHECK_VALUE(logits_in.dim() == 2, fn, ": logits must be (B, V), got ", logits_in.sizes());
  const int64_t batch = logits_in.size(0), vocab = logits_in.size(1);
  const int code = dtype_code(logits_in.scalar_type());
  TORCH_CHECK_VALUE(uniforms.dim() == 1 && uniforms.size(0) == batch, fn, ": uniforms must be (", batch, ",), got ",
                    uniforms.sizes());
  TORCH_CHECK_TYPE(uniforms.scalar_type() == at::kFloat || uniforms.scalar_type() == at::kDouble, fn,
                   ": uniforms must be float32 or float64, got ", uniforms.scalar_type());
  c10::hip::HIPGuard guard(logits_in.device().index());
  Tensor tokens = at::empty({batch}, logits_in.options().dtype(at::kLong));
  if (batch == 0) return tokens;
  const Tensor logits = logits_in.stride(1) == 1 || vocab == 1 ? logits_in : logits_in.contiguous();
  const Tensor uni = uniforms.to(logits.device()).contiguous();
  Tensor keep[4];
  const float* t = setting<float>(fn, "temperature", temperature, logits, at::kFloat, keep[0]);
  const int* k = setting<int>(fn, "top_k", top_k, logits, at::kInt, keep[1]);
  const float* p = setting<float>(fn, "top_p", top_p, logits, at::kFloat, keep[2]);
  const float* m = setting<float>(fn, "min_p", min_p, logits, at::kFloat, keep[3]);
  check(co_alibi_sample(code, logits.data_ptr(), batch == 1 ? vocab : logits.stride(0), uni.data_ptr(),
                        uni.scalar_type() == at::kDouble ? 1 : 0, t, k, p, m, temperature_all,
                        static_cast<int>(std::min<int64_t>(std::max<int64_t>(top_k_all, 0), vocab)), top_p_all, min_p_all,
                        reinterpret_cast<long long*>(tokens.data_ptr<int64_t>()), as_int(fn, "batch", batch),
                        as_int(fn, "vocab", vocab), current_stream(logits)));
  return tokens;
}

// --------------------------------------------------------------------------- autograd

// The operators called below autograd (the forward kernel) and from the backward.
std::tuple<Tensor, Tensor, Tensor> call_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& slopes,
                                            bool causal, double sm_scale, bool with_stats) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("co_alibi::fwd", "").typed<decltype(fwd_hip)>();
  return op.call(q, k, v, slopes, causal, sm_scale, with_stats);
}

// Autograd function of co_alibi::fwd (the role of the reference's CoALIBIAttention,
// co_alibi_attn.py:24-135): saves q, k, v, o, lse, stats and the slopes; lse and stats carry no
// gradient; slopes, causal, sm_scale and with_stats get none.
class FwdFunction : public torch::autograd::Function<FwdFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q,
                                                const Tensor& k, const Tensor& v, const Tensor& slopes, bool causal,
                                                double sm_scale, bool with_stats) {
    Tensor o, lse, stats;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(o, lse, stats) = call_fwd(q, k, v, slopes, causal, sm_scale, with_stats);
    }
    ctx->save_for_backward({q, k, v, o, lse, stats, slopes});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["sm_scale"] = sm_scale;
    ctx->saved_data["with_stats"] = with_stats;
    ctx->mark_non_differentiable({lse, stats});
    // lse and stats never get a gradient: without this the engine would fill zero tensors for
    // them before every backward.
    ctx->set_materialize_grads(false);
    return {o, lse, stats};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(ctx->saved_data["with_stats"].toBool(),
                "co_alibi::fwd ran with with_stats=False (inference) and has no backward");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4],
                 &stats = saved[5], &slopes = saved[6];
    const bool causal = ctx->saved_data["causal"].toBool();
    const double sm_scale = ctx->saved_data["sm_scale"].toDouble();
    const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
    Tensor dq, dk, dv;
    const Tensor& dout = grads[0];
    if (dout.defined()) {
      if (!need_k && !need_v) {
        static const auto op_dq =
            c10::Dispatcher::singleton().findSchemaOrThrow("co_alibi::bwd_dq", "").typed<decltype(bwd_dq_hip)>();
        if (need_q) dq = op_dq.call(dout, q, k, v, o, lse, stats, slopes, causal, sm_scale);
      } else {
        static const auto op =
            c10::Dispatcher::singleton().findSchemaOrThrow("co_alibi::bwd", "").typed<decltype(bwd_hip)>();
        std::tie(dq, dk, dv) = op.call(dout, q, k, v, o, lse, stats, slopes, causal, sm_scale);
        if (!need_q) dq = Tensor();
        if (!need_k) dk = Tensor();
        if (!need_v) dv = Tensor();
      }
    }
    return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> fwd_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& slopes,
                                                bool causal, double sm_scale, bool with_stats) {
  const auto r = FwdFunction::apply(q, k, v, slopes, causal, sm_scale, with_stats);
  return {r[0], r[1], r[2]};
}

// The packed form: as FwdFunction, with one saved tensor and one gradient for q, k and v.
class FwdQkvFunction : public torch::autograd::Function<FwdQkvFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& qkv,
                                                const Tensor& slopes, bool causal, double sm_scale, bool with_stats) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("co_alibi::fwd_qkv", "").typed<decltype(fwd_qkv_hip)>();
    Tensor o, lse, stats;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(o, lse, stats) = op.call(qkv, slopes, causal, sm_scale, with_stats);
    }
    ctx->save_for_backward({qkv, o, lse, stats, slopes});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["sm_scale"] = sm_scale;
    ctx->saved_data["with_stats"] = with_stats;
    ctx->mark_non_differentiable({lse, stats});
    ctx->set_materialize_grads(false);
    return {o, lse, stats};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(ctx->saved_data["with_stats"].toBool(),
                "co_alibi::fwd_qkv ran with with_stats=False (inference) and has no backward");
    const auto saved = ctx->get_saved_variables();
    Tensor dqkv;
    if (grads[0].defined() && ctx->needs_input_grad(0)) {
      static const auto op =
          c10::Dispatcher::singleton().findSchemaOrThrow("co_alibi::bwd_qkv", "").typed<decltype(bwd_qkv_hip)>();
      dqkv = op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["causal"].toBool(),
                     ctx->saved_data["sm_scale"].toDouble());
    }
    return {dqkv, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> fwd_qkv_autograd(const Tensor& qkv, const Tensor& slopes, bool causal,
                                                    double sm_scale, bool with_stats) {
  const auto r = FwdQkvFunction::apply(qkv, slopes, causal, sm_scale, with_stats);
  return {r[0], r[1], r[2]};
}

}  // namespace

TORCH_LIBRARY(co_alibi, m) {
  m.def("fwd(Tensor q, Tensor k, Tensor v, Tensor slopes, bool causal, float sm_scale, bool with_stats) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("bwd(Tensor do, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor stats, Tensor slopes, "
        "bool causal, float sm_scale) -> (Tensor, Tensor, Tensor)");
  m.def("bwd_dq(Tensor do, Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor stats, Tensor slopes, "
        "bool causal, float sm_scale) -> Tensor");
  m.def("fwd_qkv(Tensor qkv, Tensor slopes, bool causal, float sm_scale, bool with_stats) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("bwd_qkv(Tensor do, Tensor qkv, Tensor o, Tensor lse, Tensor stats, Tensor slopes, bool causal, "
        "float sm_scale) -> Tensor");
  m.def("decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor slopes, Tensor? seq_lens, SymInt max_seq_len, "
        "float sm_scale, bool with_lse) -> (Tensor, Tensor)");
  m.def("decode_tree(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor slopes, Tensor? seq_lens, "
        "Tensor? parents, Tensor? block_table, SymInt max_seq_len, float sm_scale, bool with_lse) -> (Tensor, Tensor)");
  m.def("cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor seq_lens, Tensor? counts, "
        "Tensor? rows, Tensor? block_table) -> ()");
  m.def("sample(Tensor logits, Tensor uniforms, Tensor? temperature, Tensor? top_k, Tensor? top_p, Tensor? min_p, "
        "float temperature_all, SymInt top_k_all, float top_p_all, float min_p_all) -> Tensor");
  m.def("decode_tree_8bit(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor slopes, Tensor? seq_lens, Tensor? parents, Tensor? block_table, SymInt max_seq_len, float sm_scale, "
        "bool with_lse) -> (Tensor, Tensor)");
  m.def("cache_append_8bit(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor seq_lens, Tensor? counts, Tensor? rows, Tensor? block_table) -> ()");
  m.def("cache_read_8bit(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor seq_lens, Tensor? first, "
        "Tensor? block_table, SymInt rows, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("beam_select(Tensor logits, Tensor scores, Tensor? finished, SymInt num_beams, SymInt end_token) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("cache_reorder(Tensor(a!)[] caches, Tensor block_table, Tensor pages, Tensor seq_lens, Tensor parents, "
        "SymInt page_size) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(co_alibi, CUDA, m) {
  m.impl("fwd", &fwd_hip);
  m.impl("bwd", &bwd_hip);
  m.impl("bwd_dq", &bwd_dq_hip);
  m.impl("fwd_qkv", &fwd_qkv_hip);
  m.impl("bwd_qkv", &bwd_qkv_hip);
  m.impl("decode", &decode_hip);
  m.impl("decode_tree", &decode_tree_hip);
  m.impl("cache_append", &cache_append_hip);
  m.impl("sample", &sample_hip);
  m.impl("decode_tree_8bit", &decode_tree_8bit_hip);
  m.impl("cache_append_8bit", &cache_append_8bit_hip);
  m.impl("cache_read_8bit", &cache_read_8bit_hip);
  m.impl("beam_select", &beam_select_hip);
  m.impl("cache_reorder", &cache_reorder_hip);
}

TORCH_LIBRARY_IMPL(co_alibi, Autograd, m) {
  m.impl("fwd", &fwd_autograd);
  m.impl("fwd_qkv", &fwd_qkv_autograd);
}
