"""The serving step around Co-ALiBi attention: new tokens over a cache, the cache's growth, the next token.

``co_alibi_decode_tree`` is the attention of a step's new tokens -- one, a run of them or a tree of drafts --
over a key / value cache and each other; ``co_alibi_cache_append`` writes the new (or the accepted) keys
and values behind a cache's filled rows; ``co_alibi_sample`` draws the next tokens from logits.  The first two exist over caches held in 8 bits, too
(``co_alibi_decode_tree_8bit``, ``co_alibi_cache_append_8bit``), with ``co_alibi_cache_read_8bit`` to read one back; and in
place of drawing, ``co_alibi_beam_select`` keeps the best continuations and ``co_alibi_cache_reorder`` lets a paged cache
follow them.  The reference has no counterpart of any of them.  The work runs in the gfx950 kernels of ``libco_alibi.so``
(include/co_alibi.h) through the torch operators of the same names (co_alibi_attn/ops.py).  They launch on the current stream, allocate only through torch's
caching allocator and never synchronise, so a serving step can be captured in a HIP graph.

Caches are paged or contiguous.  Paged: pools (num_pages, Hkv, page_size, D) for K and V, page_size a power of two
of at least 16, and a ``block_table`` (B, blocks) of page numbers, so that row r of sequence b is row
r % page_size of page block_table[b, r // page_size].  Contiguous (no ``block_table``): (B, Hkv, capacity, D),
as in ``co_alibi_decode``.  Index tensors are int32 (int64 ones are converted at every call).

8-bit caches: codes of one byte -- float8_e4m3fn, or int8 in [-127, 127] -- in the same layouts with dense rows, and float32
scales, one for each kv head's blocks of 16 rows: (num_pages, Hkv, page_size / 16), contiguous caches (B, Hkv,
ceil(capacity / 16)).  An element's value is code * scale.  Scales lie in [2^-40, 2^40]; a block with another one reads as NaN.
"""
from __future__ import annotations

import math

import torch

from . import _native, ops
from .co_alibi_attn import _check_head_dim, _device_slopes

__all__ = ["co_alibi_decode_tree", "co_alibi_cache_append", "co_alibi_sample", "co_alibi_decode_tree_8bit",
           "co_alibi_cache_append_8bit", "co_alibi_cache_read_8bit", "co_alibi_beam_select", "co_alibi_cache_reorder"]


def _check_new(names: str, *tensors: torch.Tensor) -> None:
    dtype = tensors[0].dtype
    for t in tensors:
        if not t.is_cuda:
            raise AssertionError("Inputs must be CUDA tensors")
        if t.dtype != dtype or dtype not in _native.DTYPE_CODES:
            raise TypeError(f"{names} must share one dtype of float32/float16/bfloat16, got "
                            + ", ".join(str(x.dtype) for x in tensors))


def _detached(t: torch.Tensor) -> torch.Tensor:
    """t without its gradient record (t itself where there is none: detaching costs the host a microsecond)."""
    return t.detach() if t.requires_grad else t


def _capacity(k_cache: torch.Tensor, block_table: torch.Tensor | None) -> int:
    """Rows a sequence's cache has room for."""
    return k_cache.shape[2] if block_table is None else block_table.shape[1] * k_cache.shape[2]


def _check_table(block_table: torch.Tensor | None, batch: int) -> None:
    if block_table is not None and (block_table.dim() != 2 or block_table.shape[0] != batch):
        raise ValueError(f"block_table must be ({batch}, blocks), got {tuple(block_table.shape)}")


def co_alibi_decode_tree(q, k, v, k_cache, v_cache, seq_len=None, parents=None, block_table=None, sm_scale=None,
                         bias_max=8.0, return_lse=False, max_seq_len=None):
    """Attention of the T newest tokens of every sequence over its cache and each other (1 <= T <= 64).

    q: (B, Hq, T, D); k, v: (B, Hkv, T, D), the new tokens' own keys and values, which the caches do not
    hold yet (``co_alibi_cache_append`` writes the ones that stay).  Strided views, such as parts of a packed
    projection, are read in place.  Caches: see the module.  ``seq_len`` is an int (every sequence; default:
    the capacity) or an integer tensor of B filled lengths on q's device, 0 allowed; then ``max_seq_len``
    (default: the capacity) bounds them, sizes the launch, and lengths outside [0, max_seq_len] are clamped.

    ``parents`` says what a token comes after: an integer tensor (T,) or (B, T) with parents[t] in [-1, t), -1
    being the cache's last row.  None is a chain, t after t - 1 (one new token; the tail of a prompt).  Token t
    sees the filled rows and its chain of parents up to itself, in that order, so its result is that of
    ``co_alibi_decode`` with the chain appended to the cache.  Any other value makes the token absent and with
    it every token after it: O = 0 and LSE = -inf there (the padding of a batch of trees).  Keys and values
    that a token does not see do not reach its result, whatever they hold; cached keys that weigh less than 2^-40
    (fp32: 2^-64) of a row's sum may be left out of it (the library's tail skip).  A sequence whose filled rows
    lie on a page outside the pool gets NaN.

    Inference only: no autograd record.  Returns o (B, Hq, T, D) in q.dtype, and with ``return_lse`` also
    the natural-log LSE (B, Hq, T) in fp32.
    """
    return _decode_tree(q, k, v, (k_cache, v_cache), None, seq_len, parents, block_table, sm_scale, bias_max, return_lse,
                        max_seq_len)


def _decode_tree(q, k, v, caches, scales, seq_len, parents, block_table, sm_scale, bias_max, return_lse, max_seq_len):
    k_cache, v_cache = caches
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q must be (B, Hq, T, D) and k, v (B, Hkv, T, D), got {tuple(q.shape)} and {tuple(k.shape)}")
    batch_size, num_heads, tokens, head_dim = q.shape
    num_kv_heads = k.shape[1]
    assert num_kv_heads >= 1 and num_heads % num_kv_heads == 0
    assert k.shape == (batch_size, num_kv_heads, tokens, head_dim)
    assert v.shape == k.shape
    if tokens > _native.MAX_TREE_TOKENS:
        raise ValueError(f"at most {_native.MAX_TREE_TOKENS} new tokens per sequence, got {tokens}")
    if scales is None:
        _check_new("q, k, v and the caches", q, k, v, k_cache, v_cache)
    else:
        _check_new("q, k and v", q, k, v)
        _check_8bit(k_cache, v_cache, *scales)
    _check_head_dim(head_dim, q.dtype, decode=True)
    _check_table(block_table, batch_size)
    capacity = _capacity(k_cache, block_table)
    lens = None
    if isinstance(seq_len, torch.Tensor):
        if seq_len.shape != (batch_size,) or seq_len.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"per-sequence lengths must be an integer tensor of shape ({batch_size},)")
        lens = seq_len
        bound = capacity if max_seq_len is None else int(max_seq_len)
        if not 0 <= bound <= capacity:
            raise ValueError(f"max_seq_len must be in [0, {capacity}], got {bound}")
    else:
        bound = capacity if seq_len is None else int(seq_len)
        if not 0 <= bound <= capacity:
            raise ValueError(f"seq_len must be in [0, {capacity}], got {bound}")
    if sm_scale is None:
        sm_scale = 1.0 / (head_dim ** 0.5)
    slopes = _device_slopes(num_heads, bias_max, q.dtype, q.device)
    if scales is None:
        o, lse = ops.decode_tree(_detached(q), _detached(k), _detached(v), _detached(k_cache), _detached(v_cache), slopes, lens,
                                 parents, block_table, bound, float(sm_scale), bool(return_lse))
    else:
        o, lse = ops.decode_tree_8bit(_detached(q), _detached(k), _detached(v), _detached(k_cache), _detached(v_cache),
                                      _detached(scales[0]), _detached(scales[1]), slopes, lens, parents, block_table, bound,
                                      float(sm_scale), bool(return_lse))
    return (o, lse) if return_lse else o


def _check_8bit(k_cache, v_cache, k_scale, v_scale) -> None:
    if not (k_cache.is_cuda and v_cache.is_cuda and k_scale.is_cuda and v_scale.is_cuda):
        raise AssertionError("Inputs must be CUDA tensors")
    fmt = k_cache.dtype
    if fmt not in _native.FORMAT_CODES or v_cache.dtype != fmt:
        raise TypeError(f"the caches must both be float8_e4m3fn or int8, got {fmt} and {v_cache.dtype}")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise TypeError(f"the scales must be float32, got {k_scale.dtype} and {v_scale.dtype}")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"k_cache and v_cache must be 4-dimensional and of one shape, got {tuple(shape)} and "
                         f"{tuple(v_cache.shape)}")
    want = (shape[0], shape[1], (shape[2] + _native.SCALE_ROWS - 1) // _native.SCALE_ROWS)
    if k_scale.shape != want or v_scale.shape != want:
        raise ValueError(f"the scales must be {want}, got {tuple(k_scale.shape)} and {tuple(v_scale.shape)}")


def co_alibi_decode_tree_8bit(q, k, v, k_cache, v_cache, k_scale, v_scale, seq_len=None, parents=None, block_table=None,
                              sm_scale=None, bias_max=8.0, return_lse=False, max_seq_len=None):
    """``co_alibi_decode_tree`` over an 8-bit cache (see the module): everything else is the same.

    The cached keys and values are code * scale, and neither q nor the weights are rounded to 8 bits: only what the cache holds
    is.  The new tokens' own k and v count as they are.  (In float16 weights of values whose block has a scale below 2^-22 (e4m3) or
    2^-25 (int8) of the largest lose bits.)  A sequence whose filled rows lie on a page outside the pool, or in a
    block whose scale is not in [2^-40, 2^40], gets NaN.
    """
    return _decode_tree(q, k, v, (k_cache, v_cache), (k_scale, v_scale), seq_len, parents, block_table, sm_scale, bias_max,
                        return_lse, max_seq_len)


def co_alibi_cache_append(k, v, k_cache, v_cache, seq_lens, block_table=None, rows=None, counts=None):
    """Writes new keys and values into the caches, in place, behind each sequence's filled rows.

    k, v: (B, Hkv, T, D), strided views included.  Row i of sequence b goes to cache row seq_lens[b] + i, for
    every i < counts[b] (integer tensor (B,); default: all), as in a padded batch of prompts.  With
    ``rows`` (integer tensor (B, n)) that row is new row rows[b, i] in place of i: the accepted path of a tree of
    drafts.  ``seq_lens`` (integer tensor (B,)) is not advanced: every layer of a model appends at the same
    place.  Counts are clamped to the rows there are; a source row outside [0, T), a cache row outside the
    capacity and a page outside the pool write nothing, and every other byte of the caches keeps its value.  The
    caches must not overlap k and v, and no two sequences may write the same row of one page.
    """
    if k.dim() != 4:
        raise ValueError(f"k and v must be (B, Hkv, T, D), got {tuple(k.shape)}")
    assert v.shape == k.shape
    _check_new("k, v and the caches", k, v, k_cache, v_cache)
    _check_head_dim(k.shape[3], k.dtype)
    _check_table(block_table, k.shape[0])
    if k_cache.requires_grad or v_cache.requires_grad:
        raise ValueError("the caches are written in place and cannot require gradients")
    ops.cache_append(_detached(k), _detached(v), k_cache, v_cache, seq_lens, counts, rows, block_table)


def co_alibi_cache_append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, seq_lens, block_table=None, rows=None, counts=None):
    """``co_alibi_cache_append`` to an 8-bit cache (see the module): the new keys and values are quantised as they are written.

    A block of 16 rows that is begun gets, for each kv head, the least power of two from 2^-40 on as its scale at which no code
    passes the format's largest (448 or 127).  A block that holds rows before ``seq_lens[b]`` keeps its scale, doubled as often as
    the new values need it, and those rows' codes are halved as often; so do a token's 16 appends leave each int8 value within one
    step of what it was, an e4m3 value within half a step of its own (near zero one smallest step).  Codes are rounded to the
    nearest, ties to even.  A value that is not finite (or past 2^40 times the largest code) makes its block's scale NaN, and so
    what is read from the block, until its first row is written again.

    Rows behind the written ones keep their bytes.  No two sequences may write the same block of one page.
    """
    if k.dim() != 4:
        raise ValueError(f"k and v must be (B, Hkv, T, D), got {tuple(k.shape)}")
    assert v.shape == k.shape
    _check_new("k and v", k, v)
    _check_8bit(k_cache, v_cache, k_scale, v_scale)
    _check_head_dim(k.shape[3], k.dtype)
    _check_table(block_table, k.shape[0])
    if any(t.requires_grad for t in (k_cache, v_cache, k_scale, v_scale)):
        raise ValueError("the caches and their scales are written in place and cannot require gradients")
    ops.cache_append_8bit(_detached(k), _detached(v), k_cache, v_cache, k_scale, v_scale, seq_lens, counts, rows, block_table)


def co_alibi_cache_read_8bit(k_cache, v_cache, k_scale, v_scale, seq_lens, rows, dtype=torch.bfloat16, block_table=None,
                             first=None):
    """Keys and values (B, Hkv, rows, D) of ``dtype`` that an 8-bit cache holds: row i is cache row ``first[b]`` + i.

    ``first`` is an integer tensor (B,) (default: 0 for all).  Rows that are not below ``seq_lens[b]`` (integer tensor (B,)) are
    zeros, rows on a page outside the pool NaN.
    """
    if dtype not in _native.DTYPE_CODES:
        raise TypeError(f"dtype must be float32/float16/bfloat16, got {dtype}")
    _check_8bit(k_cache, v_cache, k_scale, v_scale)
    _check_head_dim(k_cache.shape[3], dtype)
    if seq_lens.dim() != 1:
        raise ValueError(f"seq_lens must be (B,), got {tuple(seq_lens.shape)}")
    _check_table(block_table, seq_lens.shape[0])
    if int(rows) != rows or rows < 0:
        raise ValueError(f"rows must be a whole number >= 0, got {rows}")
    return ops.cache_read_8bit(_detached(k_cache), _detached(v_cache), _detached(k_scale), _detached(v_scale), seq_lens, first,
                               block_table, int(rows), dtype)


def co_alibi_beam_select(logits, scores, num_beams=None, finished=None, end_token=0):
    """The best continuations of a batch of beams: (scores, parents, tokens), each (B, num_beams), best first.

    logits: (B, W, V), float32, float16 or bfloat16; scores: (B, W) float32, the beams' scores so far.  A candidate is a beam w and
    a token t and scores ``scores[b, w] + log_softmax(logits[b, w])[t]``; equal scores go by beam, then by logit, then by token.
    ``num_beams`` (default W; from one beam to several at the first step) and W are at most 64, V at most 2^20.

    ``finished`` (bool (B, W)): such a beam has one candidate, ``end_token`` at its score as it is; its logits are not read.  A
    beam whose score is not finite, or whose logits hold a NaN or none above -inf, has none; neither has a logit of -inf, and
    of several +inf logits all weigh the same and the others nothing.  Places without a candidate get score -inf, parent 0 and
    token -1: no row of an embedding.

    Returns scores (float32), parents (int32) and tokens (int64).  Scores are worked out and compared in float64, from exponentials of
    float32's accuracy (so log_softmax is within 2^-22, and the same for the same logits wherever they lie), and rounded once.
    """
    if logits.dim() != 3 or not 1 <= logits.shape[2] <= _native.MAX_VOCAB or not 1 <= logits.shape[1] <= _native.MAX_BEAMS:
        raise ValueError(f"logits must be (B, W, V) with 1 <= W <= {_native.MAX_BEAMS} and 1 <= V <= {_native.MAX_VOCAB}, got "
                         f"{tuple(logits.shape)}")
    if scores.shape != logits.shape[:2]:
        raise ValueError(f"scores must be {tuple(logits.shape[:2])}, got {tuple(scores.shape)}")
    if not (logits.is_cuda and scores.is_cuda and (finished is None or finished.is_cuda)):
        raise AssertionError("Inputs must be CUDA tensors")
    if logits.dtype not in _native.DTYPE_CODES:
        raise TypeError(f"logits must be float32/float16/bfloat16, got {logits.dtype}")
    if scores.dtype != torch.float32 or (finished is not None and finished.dtype != torch.bool):
        raise TypeError("scores must be float32 and finished bool")
    n = logits.shape[1] if num_beams is None else int(num_beams)
    if not 1 <= n <= _native.MAX_BEAMS:
        raise ValueError(f"num_beams must be in [1, {_native.MAX_BEAMS}], got {n}")
    if finished is not None and (finished.shape != scores.shape or not 0 <= end_token < logits.shape[2]):
        raise ValueError(f"finished must be {tuple(scores.shape)} and end_token in [0, {logits.shape[2]}), got "
                         f"{tuple(finished.shape)} and {end_token}")
    return ops.beam_select(_detached(logits), _detached(scores), finished, n, int(end_token))


def co_alibi_cache_reorder(caches, seq_lens, parents, block_table, pages, page_size=None):
    """Lets a paged cache follow a beam selection: returns (block_table, seq_lens), new int32 tensors.

    Of B groups of W <= 64 sequences, sequence g * W + i takes over the rows of sequence g * W + ``parents[g, i]`` (integer
    tensor (B, W), clamped to [0, W)).  ``caches``: every pool (num_pages, heads, ...) under the table: all layers' keys and
    values, and the scales of 8-bit ones; dimension 2 has ``page_size`` rows (default: the first pool's size) or a divisor of
    it.  ``block_table`` (B * W, blocks): the pages in use; ``pages``, of its shape: the pages that each sequence owns, each of the
    pool's at most once -- the table that the cache began with.

    Full pages are shared by all heirs.  A page filled in part stays with its first heir; for the others its filled rows are
    copied to pages of the same column of the group's that nobody holds, and so every sequence can append.  The pools are
    written in place; what no table names any more is free and may be overwritten.  The lengths are not read by the host.
    """
    if parents.dim() != 2 or not 1 <= parents.shape[1] <= _native.MAX_BEAMS:
        raise ValueError(f"parents must be (B, W) with 1 <= W <= {_native.MAX_BEAMS}, got {tuple(parents.shape)}")
    if len(caches) == 0 or caches[0].dim() < 3:
        raise ValueError("caches must be pools (num_pages, heads, rows, ...)")
    # (The operator looks at the other pools: there may be a hundred.)
    if not (caches[0].is_cuda and seq_lens.is_cuda and parents.is_cuda and block_table.is_cuda and pages.is_cuda):
        raise AssertionError("Inputs must be CUDA tensors")
    if caches[0].requires_grad:
        raise ValueError("the caches are written in place and cannot require gradients")
    return ops.cache_reorder(caches, block_table, pages, seq_lens, parents,
                             caches[0].shape[2] if page_size is None else int(page_size))


def _setting(name, x, low, high):
    """A sampling setting as (tensor of one value per row, value of every row)."""
    if isinstance(x, torch.Tensor):
        return x, 0
    if not low <= x <= high:
        raise ValueError(f"{name} must be in [{low:g}, {high:g}], got {x}")
    return None, x


def co_alibi_sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token per row of logits (B, V), V <= 2^20, from the row's uniform number in [0, 1).

    The row's tokens in order of (logit descending, index ascending) have weights exp((logit - max) /
    temperature).  ``top_k`` keeps the first top_k of them (0: all); ``top_p`` of those the ones before which
    less than top_p of the top_k's weight lies (1: all); ``min_p`` of those the ones with at least min_p times the
    largest weight (0: all).  The first is always kept.  The token is the first, in that order, up to
    and including which more than uniform times the kept weight lies.  ``temperature`` 0 takes the first token
    (the largest logit of the lowest index).

    Each setting is a number or a tensor (B,) with one value per row (top_k integer, the others floating and taken as
    float32); values on the device cannot be checked: temperatures <= 0 or NaN take the first token, a top_k <= 0, a top_p >= 1 or NaN
    and a min_p <= 0 or NaN keep all, a top_p <= 0 and a min_p > 1 the first only, uniforms outside [0, 1) are
    taken as 0 or as the last kept token.  A row with a NaN, or with no logit above -inf, gives -1; of several
    +inf logits all have weight 1 and every other token 0.  Weights below 2^-51 of the largest
    (2^-43 at 2^20 tokens) count as 0.

    logits: float32, float16 or bfloat16; uniforms: (B,) float32 or float64.  Returns int64 tokens (B,).  The
    weights are summed exactly, so the same inputs always give the same tokens.
    """
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= _native.MAX_VOCAB:
        raise ValueError(f"logits must be (B, V) with 1 <= V <= {_native.MAX_VOCAB}, got {tuple(logits.shape)}")
    if uniforms.shape != logits.shape[:1]:
        raise ValueError(f"uniforms must be ({logits.shape[0]},), got {tuple(uniforms.shape)}")
    if not (logits.is_cuda and uniforms.is_cuda):
        raise AssertionError("Inputs must be CUDA tensors")
    if logits.dtype not in _native.DTYPE_CODES:
        raise TypeError(f"logits must be float32/float16/bfloat16, got {logits.dtype}")
    t, t_all = _setting("temperature", temperature, 0.0, math.inf)
    k, k_all = _setting("top_k", top_k, 0, math.inf)
    p, p_all = _setting("top_p", top_p, 0.0, 1.0)
    m, m_all = _setting("min_p", min_p, 0.0, 1.0)
    k_all = min(k_all, _native.MAX_VOCAB)
    if k_all != int(k_all):
        raise ValueError(f"top_k must be a whole number, got {k_all}")
    return ops.sample(_detached(logits), _detached(uniforms), t, k, p, m, float(t_all), int(k_all),
                      float(p_all), float(m_all))
