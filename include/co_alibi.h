/*
 * co_alibi.h - C ABI of the MI355X (gfx950) Co-ALiBi attention library.
 *
 * The library holds the two hot-path launches of the reference
 * (Nathancgy/Co-ALIBI) behind plain pointers and sizes:
 *
 *   co_alibi_fwd  replaces the forward launch `_co_alibi_fwd_kernel[grid](...)`
 *                 in co_alibi_attn/co_alibi_attn.py:41-57 (and the O / LSE /
 *                 RowSigTotal allocations at :35-37 move to the caller).
 *   co_alibi_bwd  replaces the backward launch `_co_alibi_bwd_kernel[grid](...)`
 *                 in co_alibi_attn/co_alibi_attn.py:101-123 together with the
 *                 dK/dV partial buffers and their reduction (:83-99, :132-133).
 *
 * a decode step the reference does not have, co_alibi_decode: its forward
 * with Sq = 1 over a key / value cache, as one split-K pass over the cache;
 * and the rest of a serving step around it, without counterparts there either:
 * co_alibi_decode_tree (several new tokens, paged caches), co_alibi_cache_append
 * and co_alibi_sample; the same over caches held in 8 bits
 * (co_alibi_decode_tree_8bit, co_alibi_cache_append_8bit,
 * co_alibi_cache_read_8bit); and beam search (co_alibi_beam_select,
 * co_alibi_cache_reorder).
 *
 * Tensor layout (except the _strided calls): contiguous row-major, q / o / dout / dq are (B, Hq, Sq, D),
 * k / v / dk / dv are (B, Hkv, Skv, D); query head h attends key/value head
 * h / (Hq / Hkv) (the head mapping of co_alibi_attn.py:143-146, done in-kernel
 * instead of by repeat_interleave).  Element type is selected by `dtype`; all
 * statistics are fp32.  `slopes` holds Hq fp32 penalty slopes (the caller
 * rounds them to the input dtype first, as co_alibi_attn.py:147 does).
 * Causal masking is top-left aligned (key j is visible to query i iff j <= i).
 *
 * Every call is asynchronous on `stream` (a hipStream_t; NULL = the null
 * stream), allocates nothing, and returns CO_ALIBI_OK or an error code; the
 * message of the last failure on the calling thread is co_alibi_last_error().
 * Pointers to element data must be 16-byte aligned, fp32 arrays 4-byte aligned.
 * Head dims 16, 32, 64, 128 and 256 in every dtype (the decode: 32 to 256, and 256 only
 * in fp16 / bf16).
 */
#ifndef CO_ALIBI_H
#define CO_ALIBI_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum co_alibi_dtype { CO_ALIBI_F32 = 0, CO_ALIBI_F16 = 1, CO_ALIBI_BF16 = 2 };

enum co_alibi_status {
  CO_ALIBI_OK = 0,
  CO_ALIBI_EINVAL = 1,       /* bad pointer, size, alignment or workspace */
  CO_ALIBI_EUNSUPPORTED = 2, /* dtype or head_dim without a kernel */
  CO_ALIBI_ELAUNCH = 3       /* the HIP runtime refused the launch */
};

/* Number of 4-byte words of the statistics `stats` that co_alibi_fwd writes beside lse and
 * co_alibi_bwd reads: 4 + B*Hq * (2 * ceil(Sq/128) + ceil(Skv/256) + ceil(Skv/64) + 2 * Sq),
 * O(B*Hq*S).  A 4-word header (flags: which work orders the forward wrote); per 128-row block
 * the first key the forward processed (int32; keys further left carry softmax weights below
 * 2^-T of their row's total, T = 26 in fp16, 32 in bf16 and 64 in fp32, and are skipped by
 * forward and backward alike; 0 when the tail skip is off); per 256-key chunk of each key head
 * the largest |k|; the order in which the kernels take their row and key blocks (int32); and
 * per row the sum of the sigmoids of the processed keys, as an fp32 hi part (B*Hq*Sq) and its
 * compensation (B*Hq*Sq).  That row sum is the reference's RowSigTotal (co_alibi_attn.py:37);
 * the backward rebuilds the penalty from it. */
size_t co_alibi_stats_numel(int batch, int heads_q, int seq_q, int seq_kv);

/* The tail skip as a library setting, for every later co_alibi_fwd and co_alibi_fwd_inference
 * call of the process: enabled != 0 (the default) leaves out the keys whose softmax weight is
 * provably below 2^-T of their row's total (above), 0 makes the forward process every key, as
 * the reference does (co_alibi_fwd_kernel.py:66-71), with no key-norm launch and no per-tile
 * test.  The backward follows what its forward recorded.  co_alibi_decode_tree, too, leaves out
 * cached keys only while it is on (its bounds are stated there).  Returns the previous setting.  No
 * counterpart in the reference, which processes every key. */
int co_alibi_set_tail_skip(int enabled);
int co_alibi_tail_skip(void);

/* Bytes of device scratch co_alibi_bwd needs (the recompute path): per-row dO.O, then per 32-key
 * block of every row the sigmoid sum from the block start on and the dA sum before it,
 * 2 * B*Hq * ceil(Skv/32) * Sq fp32 -- transient, the backward's own, where the reference holds
 * its per-query-block dK / dV partials (co_alibi_attn.py:83-99). */
size_t co_alibi_bwd_workspace_bytes(int batch, int heads_q, int seq_q, int seq_kv);

/* Bytes of device scratch that switch the backward to the score store: pass 1 keeps the
 * probabilities and score gradients of every tile it processes, 4 KB per 32 x 32 block of
 * pairs that can be visible (about 2 * Sq * Skv bytes per batch and query head when causal,
 * twice that otherwise), and pass 2 reduces them into dk and dv instead of recomputing
 * them.  0 when dtype / head_dim have no such path (fp16 and bf16 at head_dim 64 and 128
 * have it) or when (heads_q / heads_kv) * ceil(seq_q / 8192) exceeds 256.  A workspace of at
 * least this size selects the path; a smaller one (at least
 * co_alibi_bwd_workspace_bytes) the recompute path.  co_alibi_bwd_dq and co_alibi_bwd_dkdv
 * must then get the same workspace and size.  No counterpart in the reference, whose
 * backward keeps per-query-block dK / dV partials instead (co_alibi_attn.py:83-133). */
size_t co_alibi_bwd_score_store_workspace_bytes(int dtype, int batch, int heads_q, int heads_kv, int seq_q,
                                                int seq_kv, int head_dim, int causal);

/* Forward: writes o (B,Hq,Sq,D, dtype), lse (B,Hq,Sq, fp32 natural log-sum-exp
 * m_i + log(l_i), co_alibi_fwd_kernel.py:120) and stats.  The reference adds 1e-9
 * to l_i there and in the O normaliser (:115); l_i >= 1 here, so that term is
 * below fp32 resolution and is left out.  lse and stats may be NULL (inference: the
 * statistics only co_alibi_bwd reads are then not written, and every key is
 * processed); o is the same. */
int co_alibi_fwd(int dtype, const void* q, const void* k, const void* v, const float* slopes,
                 void* o, float* lse, float* stats, int batch, int heads_q, int heads_kv, int seq_q,
                 int seq_kv, int head_dim, int causal, float sm_scale, void* stream);

/* Forward for inference with the tail skip: o only (no lse or stats), skipping the keys
 * whose softmax weight is below 2^-T of the row total as co_alibi_fwd does with its
 * statistics (co_alibi_fwd with lse = stats = NULL computes every key).  workspace holds
 * co_alibi_fwd_inference_workspace_bytes(...) bytes (256-byte aligned): the largest |k|
 * per 256-key chunk of every key head and the order of the row blocks.  No counterpart in
 * the reference, whose forward always saves its statistics (co_alibi_attn.py:35-57). */
size_t co_alibi_fwd_inference_workspace_bytes(int batch, int heads_q, int seq_q, int seq_kv);
int co_alibi_fwd_inference(int dtype, const void* q, const void* k, const void* v, const float* slopes,
                           void* o, void* workspace, size_t workspace_bytes, int batch, int heads_q,
                           int heads_kv, int seq_q, int seq_kv, int head_dim, int causal, float sm_scale,
                           void* stream);

/* Forward on operands in other layouts, as a model's projections leave them ((B, S, H, D) memory,
 * parts of a packed QKV tensor): strides holds the batch, head and row strides in elements of q, k, v
 * and o, in this order (12 values).  A row's head_dim elements are consecutive; strides are whole
 * 16-byte units, row strides at least head_dim and at most 2^20, k's and v's the same.  An output's rows
 * must not overlap: of its dimensions longer than 1, in order of their strides, each steps past all that
 * the smaller ones cover.  With stats it is co_alibi_fwd; without (NULL) it is
 * co_alibi_fwd_inference, with its workspace.  lse and stats keep their layouts.
 * The reference's kernels take the strides of q, k, v and o too (co_alibi_attn.py:41-57). */
int co_alibi_fwd_strided(int dtype, const void* q, const void* k, const void* v, const float* slopes, void* o,
                         const long long* strides, float* lse, float* stats, void* workspace,
                         size_t workspace_bytes, int batch, int heads_q, int heads_kv, int seq_q, int seq_kv,
                         int head_dim, int causal, float sm_scale, void* stream);

/* Backward: given dout and the forward's q, k, v, o, lse, stats, writes dq
 * (B,Hq,Sq,D), dk and dv (B,Hkv,Skv,D), all in dtype.  For Hkv < Hq the key /
 * value gradients are summed over the query heads of each group.  workspace
 * must hold co_alibi_bwd_workspace_bytes(...) bytes (256-byte aligned). */
int co_alibi_bwd(int dtype, const void* dout, const void* q, const void* k, const void* v,
                 const void* o, const float* lse, const float* stats, const float* slopes, void* dq,
                 void* dk, void* dv, void* workspace, size_t workspace_bytes, int batch, int heads_q,
                 int heads_kv, int seq_q, int seq_kv, int head_dim, int causal, float sm_scale,
                 void* stream);

/* co_alibi_bwd on operands in other layouts (co_alibi_fwd_strided's rules): strides holds those of
 * dout, q, k, v, o, dq, dk and dv, in this order (24 values).  On the score-store path only: a smaller
 * workspace than co_alibi_bwd_score_store_workspace_bytes(...) is CO_ALIBI_EINVAL. */
int co_alibi_bwd_strided(int dtype, const void* dout, const void* q, const void* k, const void* v,
                         const void* o, const float* lse, const float* stats, const float* slopes, void* dq,
                         void* dk, void* dv, const long long* strides, void* workspace, size_t workspace_bytes,
                         int batch, int heads_q, int heads_kv, int seq_q, int seq_kv, int head_dim, int causal,
                         float sm_scale, void* stream);

/* The two passes of co_alibi_bwd as separate calls, for callers that time or
 * schedule them apart.  co_alibi_bwd_dq writes dq and fills the workspace
 * (per-row dO.O and the per-32-key-block sums, or the score store); co_alibi_bwd_dkdv
 * then writes dk and dv from that workspace.  Issued in this order on one
 * stream they are exactly co_alibi_bwd.  The reference runs both in one
 * kernel (co_alibi_attn/co_alibi_bwd_kernel.py:17-146). */
int co_alibi_bwd_dq(int dtype, const void* dout, const void* q, const void* k, const void* v,
                    const void* o, const float* lse, const float* stats, const float* slopes, void* dq,
                    void* workspace, size_t workspace_bytes, int batch, int heads_q, int heads_kv,
                    int seq_q, int seq_kv, int head_dim, int causal, float sm_scale, void* stream);

int co_alibi_bwd_dkdv(int dtype, const void* dout, const void* q, const void* k, const void* v,
                      const float* lse, const float* stats, const float* slopes, void* dk, void* dv,
                      void* workspace, size_t workspace_bytes, int batch, int heads_q, int heads_kv,
                      int seq_q, int seq_kv, int head_dim, int causal, float sm_scale, void* stream);

/* Which kernel forms calls of this shape take under the current tail-skip setting, or -1 for an
 * unsupported one: on small grids the forward and backward pass 1 split a row block over four
 * work-groups (which rounds sums in another order), the forward also the longer half of the row blocks on
 * middle grids, the fp32 forward at head dim 64 has two register budgets, and the recompute path's pass 2
 * works on 32 keys per work-group.  No counterpart in the reference; it serves tests and measurements. */
#define CO_ALIBI_FORM_FWD_SPLIT 1
#define CO_ALIBI_FORM_FWD_LONG_ROWS 2
#define CO_ALIBI_FORM_DQ_SPLIT 4
#define CO_ALIBI_FORM_DKDV_KEYS 8
#define CO_ALIBI_FORM_FWD_ROOMY 16
int co_alibi_attention_forms(int dtype, int batch, int heads_q, int heads_kv, int seq_q, int seq_kv,
                             int head_dim, int causal);

/* Bytes of device scratch co_alibi_decode needs: the split-K partials, 4 + head_dim
 * fp32 per (batch, query head, split), for min(ceil(seq_kv / 128), 1024) splits (each
 * split walks one or more 128-key chunks of the cache). */
size_t co_alibi_decode_workspace_bytes(int batch, int heads_q, int seq_kv, int head_dim);

/* How a decode of this shape is launched: the splits of every sequence, each a work-group per key
 * head (1: no partials and no merge launch).  With per-sequence lengths (ragged != 0) a negative
 * value: the lengths decide, in place of that many by the bound seq_kv.  No counterpart in the
 * reference; it serves tests and measurements. */
int co_alibi_decode_splits(int dtype, int batch, int heads_kv, int seq_kv, int head_dim, int ragged);

/* Decode: one new query per (batch, query head) against a key / value cache.
 * q and o are (B, Hq, D); k_cache and v_cache are (B, Hkv, kv_capacity, D).  Sequence
 * b has its first len_b rows of every head filled, all of them visible to the query
 * (the newest position): len_b = seq_lens[b] when seq_lens (B int32 on the device) is
 * given, clamped to [0, seq_kv] in the kernel, else seq_kv.  A sequence of length 0
 * gets O = 0 and LSE = -inf.  lse (B*Hq fp32, natural log) may be NULL.  The
 * reference has no decode entry point: this is its forward, co_alibi_attention(q, k,
 * v, causal=False) (co_alibi_attn/co_alibi_attn.py:137-148), with Sq = 1 and the
 * caches cut to len_b rows; its top-left causal mask (co_alibi_fwd_kernel.py:80-90)
 * would show an Sq = 1 query only the first key.  Head dims 32 to 256 (256 in fp16 /
 * bf16 only); at most 32 query heads per kv head, seq_kv <= 2^21 (it sizes the grid and the workspace); workspace holds
 * co_alibi_decode_workspace_bytes(...) bytes (256-byte aligned). */
int co_alibi_decode(int dtype, const void* q, const void* k_cache, const void* v_cache,
                    const float* slopes, const int* seq_lens, void* o, float* lse,
                    void* workspace, size_t workspace_bytes, int batch, int heads_q, int heads_kv,
                    int seq_kv, int kv_capacity, int head_dim, float sm_scale, void* stream);

/* co_alibi_decode for callers that cannot allocate device memory (work captured into a HIP
 * graph, tight serving loops, harnesses that forbid hipMalloc).  It has no counterpart in the
 * reference.  Arguments are those of co_alibi_decode without the workspace: the split-K
 * partials go to a buffer of CO_ALIBI_DECODE_SCRATCH_BYTES that the library holds on every GPU
 * it runs on until the process ends, laid out for this launch's split count ((4 + head_dim)
 * fp32 per (batch, query head, split), each of the three per-split arrays 256-byte aligned).  A
 * decode whose partials exceed it returns CO_ALIBI_EINVAL.  The call allocates nothing.  All
 * calls on one GPU share its buffer, which keeps the last call's contents: calls that overlap on
 * one GPU (for instance on two streams) race, so order them on one stream. */
#define CO_ALIBI_DECODE_SCRATCH_BYTES (32u << 20)
int co_alibi_decode_noalloc(int dtype, const void* q, const void* k_cache, const void* v_cache,
                            const float* slopes, const int* seq_lens, void* o, float* lse, int batch,
                            int heads_q, int heads_kv, int seq_kv, int kv_capacity, int head_dim,
                            float sm_scale, void* stream);

/* The calls below take key / value caches as pages or as one contiguous cache per sequence.  With a
 * block_table (batch x blocks_per_seq int32 on the device) the caches are pools of num_pages pages (page,
 * heads_kv, page_size, head_dim), page_size a power of two >= 16, and cache row r of sequence b is row
 * r % page_size of page block_table[b][r / page_size].  Without one (NULL) they are (batch, heads_kv,
 * page_size, head_dim), page_size being the capacity, and blocks_per_seq and num_pages are not read.  Strides
 * follow co_alibi_fwd_strided's rules (k and v may differ), from page to page in place of the batch stride;
 * NULL: everything is contiguous. */

/* Tree decode: the attention of `tokens` new tokens per sequence (1 to 64) over a cache and each other.
 * q and o are (B, Hq, tokens, D), o contiguous; k and v (B, Hkv, tokens, D) are the new tokens' own keys and
 * values, which the cache does not hold yet.  Token t sees the sequence's filled rows and, after them, its
 * chain of parents up to itself: parents (int32 on the device; tokens values for every sequence, or with
 * parents_per_seq != 0 batch x tokens) holds in [-1, t) the token that t comes after, -1 for the cache's last
 * row.  NULL is a chain: t after t - 1.  Any other value makes the token absent, and every token whose
 * chain meets it: o = 0 and lse = -inf there.  The result for token t is co_alibi_decode's for its query with
 * the chain's keys and values appended to the cache.  Filled rows: seq_lens (B int32 on the device) clamped to
 * [0, seq_kv], or NULL for seq_kv (>= 0).  A sequence whose filled rows lie on a page outside the pool gets
 * NaN.  Rows past the filled ones, pages that hold none, and keys and values of tokens outside a token's chain
 * do not reach its result whatever they hold.  With the tail skip on, cached keys that weigh less than 2^-40
 * (fp32: 2^-64) of a row's sum may be left out of it; with it off every filled row is read.  Head dims 16 to 256 (256 in fp16 / bf16 only).  strides: those
 * of q, k, v, k_cache and v_cache (15 values) or NULL.  workspace holds
 * co_alibi_decode_tree_workspace_bytes(...) bytes (256-byte aligned; may be NULL when that is 0, as it also is for a
 * shape that the call refuses). */
size_t co_alibi_decode_tree_workspace_bytes(int dtype, int batch, int heads_q, int heads_kv, int tokens, int seq_kv,
                                            int head_dim);
int co_alibi_decode_tree(int dtype, const void* q, const void* k, const void* v, const void* k_cache,
                         const void* v_cache, const long long* strides, const float* slopes, const int* seq_lens,
                         const int* parents, int parents_per_seq, const int* block_table, int blocks_per_seq,
                         int num_pages, int page_size, void* o, float* lse, void* workspace, size_t workspace_bytes,
                         int batch, int heads_q, int heads_kv, int tokens, int seq_kv, int head_dim, float sm_scale,
                         void* stream);

/* Cache append: writes new keys and values (k, v: (B, Hkv, tokens, D)) into the caches behind each sequence's
 * filled rows.  Row i of sequence b, for i < counts[b] (B int32, or NULL: new_rows), is new row rows[b][i]
 * (batch x new_rows int32, or NULL: row i) and goes to cache row seq_lens[b] + i.  seq_lens itself is the
 * caller's to advance.  Counts are clamped to [0, new_rows]; a source row outside [0, tokens), a cache row
 * outside the capacity and a page outside the pool write nothing.  Every other byte of the caches keeps its
 * value.  The caches must not overlap k and v, and no two sequences may write one page's same row.
 * strides: those of k, v, k_cache and v_cache (12 values) or NULL. */
int co_alibi_cache_append(int dtype, const void* k, const void* v, void* k_cache, void* v_cache,
                          const long long* strides, const int* seq_lens, const int* counts, const int* rows,
                          int new_rows, const int* block_table, int blocks_per_seq, int num_pages, int page_size,
                          int batch, int heads_kv, int tokens, int head_dim, void* stream);

/* Sampling: one token per row of logits (batch rows of vocab elements, row_stride elements apart; element
 * aligned; vocab at most 2^20).  With a row's tokens in order (logit descending, then index ascending) and
 * weights exp((logit - max) / temperature): top_k keeps the first top_k (<= 0: all); top_p of those the ones
 * before which less than top_p times the top_k's total weight lies (>= 1: all); min_p of those the ones of
 * weight >= min_p (<= 0: all).  The first token is always kept.  The result is the first token in that order
 * whose inclusive weight sum exceeds uniform times the kept sum (uniforms: batch fp32, or fp64 with
 * uniforms_f64 != 0, in [0, 1); values outside are taken as 0 or as the last kept token).  temperature <= 0
 * takes the first token.  A row with a NaN, or with no logit above -inf, gives -1.  Of several +inf logits all have
 * weight 1 and the others 0.  temperature, top_k, top_p and min_p are arrays of one value per row on the
 * device, or NULL: then the _all value is every row's.  Weights are summed exactly in integers, so a call's
 * result does not depend on the order of its sums. */
int co_alibi_sample(int dtype, const void* logits, long long row_stride, const void* uniforms, int uniforms_f64,
                    const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                    double temperature_all, int top_k_all, double top_p_all, double min_p_all, long long* tokens,
                    int batch, int vocab, void* stream);

/* Caches held in 8 bits: an element is a code (format CO_ALIBI_E4M3: e4m3 without infinities, largest 448; CO_ALIBI_INT8: a
 * two's complement byte, written in [-127, 127]) and its value code * scale, with one fp32 scale for each kv head's blocks of 16
 * rows: k_scale and v_scale are (num_pages, heads_kv, page_size / 16), or (batch, heads_kv, ceil(page_size / 16)) without a
 * block_table.  scale_strides holds their strides from page (sequence) to page and head to head, k_scale's then v_scale's, or is
 * NULL: contiguous; a head's scales follow one another.  Cache strides are in elements, whole 16-byte units, with the row stride
 * head_dim.  Scales must lie in [2^-40, 2^40]; a block with another one (a NaN among them) reads as NaN. */
enum co_alibi_format { CO_ALIBI_E4M3 = 0, CO_ALIBI_INT8 = 1 };

/* co_alibi_cache_append to an 8-bit cache.  A block that is begun gets the least power of two from 2^-40 on at which no new
 * value's code passes the largest; a block that holds rows before seq_lens[b] keeps its scale, doubled as often as the new values
 * need, and the codes of those rows are halved as often.  Codes are rounded to the nearest, ties to even.  A new value that is not
 * finite, or needs a scale past 2^40, makes its block's scale NaN, until the block's first row is written again.  No two
 * sequences may write one page's same block.  strides: those of k, v, k_cache and v_cache (12 values) or NULL. */
int co_alibi_cache_append_8bit(int dtype, int format, const void* k, const void* v, void* k_cache, void* v_cache,
                               float* k_scale, float* v_scale, const long long* strides, const long long* scale_strides,
                               const int* seq_lens, const int* counts, const int* rows, int new_rows, const int* block_table,
                               int blocks_per_seq, int num_pages, int page_size, int batch, int heads_kv, int tokens,
                               int head_dim, void* stream);

/* Rows of an 8-bit cache as values of `dtype`: k and v (batch, heads_kv, rows, D), contiguous, get cache row first[b] + i
 * (batch int32, or NULL: i) of sequence b in row i: zeros where it is not below seq_lens[b], NaN on a page outside the pool.
 * strides: those of k_cache and v_cache (6 values) or NULL. */
int co_alibi_cache_read_8bit(int dtype, int format, const void* k_cache, const void* v_cache, const float* k_scale,
                             const float* v_scale, const long long* strides, const long long* scale_strides,
                             const int* seq_lens, const int* first, int rows, const int* block_table, int blocks_per_seq,
                             int num_pages, int page_size, void* k, void* v, int batch, int heads_kv, int head_dim,
                             void* stream);

/* co_alibi_decode_tree over an 8-bit cache: q, k, v and o stay in `dtype`, the cached keys and values are code * scale in fp32.
 * A sequence with a filled block whose scale is not in [2^-40, 2^40] gets NaN. */
size_t co_alibi_decode_tree_8bit_workspace_bytes(int dtype, int batch, int heads_q, int heads_kv, int tokens, int seq_kv,
                                                 int head_dim);
int co_alibi_decode_tree_8bit(int dtype, int format, const void* q, const void* k, const void* v, const void* k_cache,
                              const void* v_cache, const float* k_scale, const float* v_scale, const long long* strides,
                              const long long* scale_strides, const float* slopes, const int* seq_lens, const int* parents,
                              int parents_per_seq, const int* block_table, int blocks_per_seq, int num_pages, int page_size,
                              void* o, float* lse, void* workspace, size_t workspace_bytes, int batch, int heads_q,
                              int heads_kv, int tokens, int seq_kv, int head_dim, float sm_scale, void* stream);

/* Beam selection: of every sequence's candidates (w, t), beam w < beams continued with token t < vocab, the num_beams with the
 * largest score, scores[b][w] + log_softmax(logits[b][w])[t], best first; equal scores go by beam, then by logit, then by token.
 * Scores are compared in fp64 and rounded once; log_softmax is within 2^-22, and the same for the same logits wherever they lie.
 * logits: (batch, beams, vocab) in `dtype`, strides its batch and beam strides in elements (2 values) or NULL: contiguous.
 * scores: (batch, beams) fp32.  A beam with finished[b][w] != 0 (batch x beams bytes, or NULL) has one candidate, end_token at its
 * score as it is, and its logits are not read.  A beam whose score is not finite, whose logits hold a NaN or none above -inf
 * has no candidates, and a logit of -inf is none; of +inf logits all weigh the same and every other one nothing.  Results, each
 * (batch, num_beams): out_scores, parents (the beam) and tokens; places without a candidate get -inf, 0 and -1.  At most 64 beams in
 * and out, vocab <= 2^20.  workspace holds co_alibi_beam_select_workspace_bytes(...) bytes (256-byte aligned). */
size_t co_alibi_beam_select_workspace_bytes(int dtype, int batch, int beams, int num_beams, int vocab);
int co_alibi_beam_select(int dtype, const void* logits, const long long* strides, const float* scores,
                         const unsigned char* finished, int end_token, float* out_scores, int* parents, long long* tokens,
                         void* workspace, size_t workspace_bytes, int batch, int beams, int num_beams, int vocab,
                         void* stream);

/* Cache reorder: sequence g * beams + i of a paged cache takes over the rows of sequence g * beams + parents[g][i] (batch x beams
 * int32, clamped to [0, beams)).  block_table and pages are (batch * beams, blocks_per_seq): the pages in use, and the ones that
 * each sequence owns, every page of the pool at most once among them; the entries of a group's column in block_table are
 * entries of that column in pages.  Full pages are shared.  A page that is filled in part stays with its first heir and is copied
 * for the others, its filled rows only, into pages of the group's column that nobody holds; columns behind the filled rows
 * get such pages, too.  So a page that is filled in part belongs to one sequence, which co_alibi_cache_append needs.
 * out_table and out_lens (batch * beams) receive the new table and lengths (they must not overlap the inputs); the pools, num_pools
 * of them, are written in place.  shapes has five values for each: bytes from page to page, and head to head, heads, entries per
 * page and head, bytes of an entry; entries follow one another and stand for page_size / entries rows each.  Everything is in
 * whole 4 bytes.  Copies to or from a page outside [0, num_pages) are left out.  At most 64 beams. */
int co_alibi_cache_reorder(void* const* pools, const long long* shapes, int num_pools, const int* block_table,
                           const int* pages, const int* seq_lens, const int* parents, int* out_table, int* out_lens,
                           int batch, int beams, int blocks_per_seq, int num_pages, int page_size, void* stream);

/* Measurement helper with no counterpart in the reference: `blocks` work-groups of 256
 * threads each issue `iters` rounds of four independent fp16 32x32x16 MFMAs per
 * wavefront.  ticks (2*blocks uint64) receives, per work-group, the shader-clock and the
 * 100 MHz real-time counter deltas around the loop; sink (256*blocks fp32) receives a
 * checksum.  The benchmark derives the sustained clock and MFMA rate from it. */
int co_alibi_probe_mfma(void* ticks, void* sink, int blocks, int iters, void* stream);

/* Message describing the last failed call on this thread ("" if none). */
const char* co_alibi_last_error(void);

/* ABI version of this header: 6 (O(S) statistics, the row sigmoid sums in place of the
 * per-block penalty sums; the tail-skip setting). */
int co_alibi_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* CO_ALIBI_H */
