"""co_alibi_decode_tree against the float64 oracle (oracle/serving.py).  Needs an MI355X.

Tolerances: the oracle's first-order bound of what fp32 arithmetic and the rounding of the weights to the
input type can change, plus half a step of the output type.
"""
import math

import pytest
import torch

from co_alibi_attn import _native, co_alibi_attention, co_alibi_cache_append, co_alibi_decode, co_alibi_decode_tree
from oracle import co_alibi_ref as ref
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAME = {F16: "fp16", BF16: "bf16", F32: "fp32"}


def random_parents(B, T, gen, absent=False):
    par = torch.stack([torch.arange(T) - torch.randint(1, 6, (T,), generator=gen) for _ in range(B)]).clamp_(min=-1)
    if absent:  # a node of its own as parent, a later one, one below -1: each takes its descendants with it
        for b in range(B):
            for bad in (lambda t: t, lambda t: t + 1, lambda t: -2, lambda t: 1 << 30):
                t = int(torch.randint(0, T, (1,), generator=gen))
                par[b, t] = bad(t)
    return par.to(torch.int32)


def make(B, Hq, Hkv, T, lens, D, dtype, page, seed=0, scale=0.5, garbage=math.nan):
    """Inputs on the CPU.  Rows no sequence has filled, and pages no sequence uses, hold garbage."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: (torch.randn(*s, generator=gen) * scale).to(dtype)  # noqa: E731
    q, k, v = n(B, Hq, T, D), n(B, Hkv, T, D), n(B, Hkv, T, D)
    rows = max(max(lens), 1)
    if page == 0:
        kc, vc, table = n(B, Hkv, rows + 3, D), n(B, Hkv, rows + 3, D), None
        for b in range(B):
            kc[b, :, lens[b]:] = garbage
            vc[b, :, lens[b]:] = garbage
        return q, k, v, kc, vc, table
    blocks = -(-rows // page)
    order = torch.randperm(B * blocks + 2, generator=gen)
    table = order[:B * blocks].view(B, blocks).to(torch.int32)
    kc, vc = n(B * blocks + 2, Hkv, page, D), n(B * blocks + 2, Hkv, page, D)
    used = torch.zeros(B * blocks + 2, page, dtype=torch.bool)
    for b in range(B):
        for r in range(lens[b]):
            used[table[b, r // page], r % page] = True
        table[b, -(-lens[b] // page):] = -7  # entries past the filled rows are never read
    kc.masked_fill_(~used[:, None, :, None], garbage)
    vc.masked_fill_(~used[:, None, :, None], garbage)
    return q, k, v, kc, vc, table


def run(q, k, v, kc, vc, table, lens, parents, **kw):
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    o, lse = co_alibi_decode_tree(dev(q), dev(k), dev(v), dev(kc), dev(vc), parents=dev(parents), block_table=dev(table),
                                  seq_len=torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True, **kw)
    torch.cuda.synchronize()
    return o.cpu(), lse.cpu()


def lam_of(Hq, dtype, bias_max=8.0):
    return ref.slopes(Hq, bias_max, dtype=dtype).float()


def check(got, want, dtype):
    o, lse = got
    ro, rlse, ob, lb = want
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny if dtype == F16 else 0.0  # fp16 steps are 2^-24 below its normals
    assert o.dtype == dtype and torch.isfinite(o).all()
    over = (o.double() - ro).abs() - (half * (ro.abs() + ob) + ob + tiny * half)
    print(f"  o: max err {(o.double() - ro).abs().max():.2e}, worst margin {over.max():.2e}", flush=True)
    assert over.max() <= 0
    empty = torch.isneginf(rlse)
    assert torch.equal(torch.isneginf(lse), empty)
    err = torch.where(empty, torch.zeros_like(rlse), (lse.double() - rlse).abs() - lb)
    assert err.max() <= 0, f"lse off by {err.max():.2e} beyond its bound"


# (B, Hq, Hkv, T, lens, D, page)
CASES = [
    (1, 4, 4, 1, [0], 64, 0),               # nothing cached: the token sees itself
    (1, 4, 4, 1, [1], 64, 64),
    (2, 8, 2, 1, [300, 0], 128, 16),        # one token, 4 heads a group, an empty cache beside
    (3, 6, 2, 5, [127, 128, 129], 32, 32),  # around a 128-key chunk; 15 rows
    (2, 12, 12, 7, [33, 500], 64, 0),
    (1, 8, 1, 4, [257], 128, 64),           # 32 rows
    (1, 11, 1, 3, [100], 64, 16),           # 33
    (2, 8, 2, 16, [31, 640], 128, 64),      # 64
    (1, 5, 1, 13, [211], 64, 32),           # 65
    (1, 4, 1, 33, [97], 128, 16),           # 132
    (2, 4, 2, 64, [70, 5], 16, 16),         # every new token there can be; 128 rows; head dim 16
    (1, 2, 2, 63, [40], 128, 256),
    (1, 32, 1, 2, [130], 64, 64),           # 32 heads a group
    (1, 40, 1, 1, [130], 32, 16),           # more than the single-token decode takes
    (1, 4, 4, 1, [1500], 64, 64),           # merged from splits at every head dim
    (3, 6, 2, 5, [900, 640, 0], 32, 32),
    (2, 4, 2, 7, [70, 1000], 16, 16),
    (2, 3, 3, 2, [511, 513], 64, 16),       # five chunks and six
]


@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=NAME.get)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "B{}_Hq{}_Hkv{}_T{}_L{}_D{}_p{}".format(*c[:4], max(c[4]), *c[5:]))
def test_tree_matches_oracle(case, dtype):
    B, Hq, Hkv, T, lens, D, page = case
    inputs = make(*case[:6], dtype, page, seed=T + max(lens))
    gen = torch.Generator().manual_seed(T)
    for parents in (None, random_parents(B, T, gen, absent=T > 4)):
        print(case, NAME[dtype], "chain" if parents is None else "tree", flush=True)
        want = oracle.decode_tree(*inputs[:5], lens, parents, inputs[5], lam_of(Hq, dtype), D ** -0.5)
        check(run(*inputs, lens, parents), want, dtype)


@pytest.mark.parametrize("dtype", (BF16, F16), ids=NAME.get)
@pytest.mark.parametrize("case", [(1, 8, 2, 1, [300], 256, 64), (2, 4, 1, 20, [129, 1], 256, 16)], ids=str)
def test_tree_head_dim_256(case, dtype):
    test_tree_matches_oracle(case, dtype)


@pytest.mark.parametrize("seed", range(12))
def test_tree_random(seed):
    gen = torch.Generator().manual_seed(100 + seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))  # noqa: E731
    B, Hkv, G, T = r(1, 4), r(1, 3), r(1, 8), r(1, 64)
    D = (16, 32, 64, 128, 256)[r(0, 4)]
    dtype = (F16, BF16, F32 if D < 256 else BF16)[r(0, 2)]
    page = (0, 16, 32, 64, 128)[r(0, 4)]
    lens = [r(0, 400) for _ in range(B)]
    print(seed, B, G * Hkv, Hkv, T, lens, D, page, NAME[dtype], flush=True)
    inputs = make(B, G * Hkv, Hkv, T, lens, D, dtype, page, seed=seed, scale=(0.3, 1.0, 2.0)[r(0, 2)])
    parents = random_parents(B, T, gen, absent=r(0, 1) == 1)
    want = oracle.decode_tree(*inputs[:5], lens, parents, inputs[5], lam_of(G * Hkv, dtype), D ** -0.5)
    check(run(*inputs, lens, parents), want, dtype)


def few_long(B, long, seed):
    """Lengths around `long` at a few places, else up to 90, with 0 and 1 among them."""
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(2, 91, (B,), generator=gen)
    lens[0], lens[B // 2], lens[B - 1], lens[1], lens[B - 2] = long, long - 37, long // 3, 0, 1
    return lens.tolist()


# Enough sequences and rows that the launch divides its splits by the sequences' own lengths.
RAGGED = [
    (16, 8, 8, 2, few_long(16, 2305, 1), 128, 64, BF16),    # 16-row blocks
    (24, 16, 4, 10, few_long(24, 2900, 2), 128, 16, F16),   # 64
    (40, 32, 2, 5, few_long(40, 1793, 3), 128, 32, BF16),   # 128, of which 80 rows are used
    (30, 16, 1, 10, few_long(30, 3000, 4), 64, 64, F16),    # two blocks
    (100, 2, 1, 1, few_long(100, 4200, 5), 64, 0, BF16),    # more sequences than a wavefront's lanes
    (20, 4, 4, 3, few_long(20, 1700, 6), 128, 64, F32),
    (30, 2, 2, 2, few_long(30, 2400, 7), 256, 64, BF16),
]


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: "B{}_Hq{}_Hkv{}_T{}_L{}_D{}_p{}_{}".format(
    *c[:4], max(c[4]), *c[5:7], NAME[c[7]]))
def test_tree_ragged_batch(case):
    B, Hq, Hkv, T, lens, D, page, dtype = case
    inputs = make(*case[:6], dtype, page, seed=B)
    parents = random_parents(B, T, torch.Generator().manual_seed(B), absent=T > 4)
    want = oracle.decode_tree(*inputs[:5], lens, parents, inputs[5], lam_of(Hq, dtype), D ** -0.5)
    check(run(*inputs, lens, parents), want, dtype)
    check(run(*inputs, lens, parents, max_seq_len=max(lens)), want, dtype)


@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=NAME.get)
def test_old_keys_of_large_scores_count(dtype):
    """Old keys fade below what a sum shows and are left out of it, but not one whose score makes up for its age."""
    B, Hq, Hkv, T, L, D = 1, 8, 1, 12, 5000, 128
    q, k, v, kc, vc, table = make(B, Hq, Hkv, T, [L], D, dtype, 64, seed=31)
    lam = lam_of(Hq, dtype)

    def want():
        return oracle.decode_tree(q, k, v, kc, vc, [L], None, table, lam, D ** -0.5)

    plain = want()
    check(run(q, k, v, kc, vc, table, [L], None), plain, dtype)
    for row in (700, 3000):  # as much as nodes 0 and 5 of the flattest head, and of the fourth, can ask for
        for h, t in ((7, 0), (3, 5)):
            kc[table[0, row // 64], :, row % 64] = (8 * q[0, h, t].float()).to(dtype)
            planted = want()
            check(run(q, k, v, kc, vc, table, [L], None), planted, dtype)
            if h == 7:
                assert (planted[0][0, h, t] - plain[0][0, h, t]).abs().max() > 0.01  # ten times what roundings may do here
    with _native.tail_skip(False):
        check(run(q, k, v, kc, vc, table, [L], None), planted, dtype)
    kc[table[0, 1], 0, 3, 5] = math.nan  # a key that every row sees
    o, lse = run(q, k, v, kc, vc, table, [L], None)
    assert o.isnan().all() and lse.isnan().all()


def test_ragged_batch_with_a_page_outside_the_pool():
    B, lens = 16, few_long(16, 2305, 8)
    q, k, v, kc, vc, table = make(B, 8, 8, 2, lens, 128, BF16, 64, seed=8)
    sound, _ = run(q, k, v, kc, vc, table, lens, None)
    table[0, 20], table[3, 0] = kc.shape[0], -1
    got, lse = run(q, k, v, kc, vc, table, lens, None)
    for b in range(B):
        if b in (0, 3):
            assert got[b].isnan().all() and lse[b].isnan().all()
        else:
            assert torch.equal(got[b], sound[b])


def test_ragged_batches_in_every_order_of_sequences():
    """The same sequences in another order, or with others' lengths changed: the long one's result moves by rounding only."""
    B, Hq, Hkv, T, D = 16, 8, 8, 2, 128
    lens = few_long(B, 2305, 9)
    q, k, v, kc, vc, table = make(B, Hq, Hkv, T, lens, D, F16, 64, seed=9)
    want = oracle.decode_tree(q, k, v, kc, vc, lens, None, table, lam_of(Hq, F16), D ** -0.5)
    for seed in range(3):
        order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
        got = run(q[order], k[order], v[order], kc, vc, table[order], [lens[b] for b in order], None)
        check(got, tuple(w[order] for w in want), F16)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", (BF16, F32), ids=NAME.get)
def test_unseen_tokens_do_not_reach_a_result(dtype, bad):
    """Keys and values of another branch hold infinities and NaN; so do those of an absent node."""
    B, Hq, Hkv, T, D = 1, 8, 2, 12, 64
    parents = torch.tensor([[-1, 0, 0, 1, 2, 3, 4, 5, -2, 8, 6, 7]], dtype=torch.int32)
    q, k, v, kc, vc, table = make(B, Hq, Hkv, T, [150], D, dtype, 16, seed=5)
    clean = oracle.decode_tree(q, k, v, kc, vc, [150], parents, table, lam_of(Hq, dtype), D ** -0.5)
    k[:, :, 8] = v[:, :, 8] = bad                # absent
    k[0, 0, 2, 3] = v[0, 1, 2, 7] = bad          # the branch 2, 4, 6, 10
    o, lse = run(q, k, v, kc, vc, table, [150], parents)
    keep = [0, 1, 3, 5, 7, 8, 9, 11]
    check((o[:, :, keep], lse[:, :, keep]), tuple(x[:, :, keep] for x in clean), dtype)
    hit = [2, 4, 6, 10]
    assert not torch.isfinite(o[0, 4:, hit, 7]).any()    # the value's own column, for the heads of its kv head
    others = [d for d in range(D) if d != 7]
    check((o[:, 4:][:, :, hit][..., others], lse[:, 4:][:, :, hit]),
          tuple(x[:, 4:][:, :, hit][..., others] if x.dim() == 4 else x[:, 4:][:, :, hit] for x in clean), dtype)


def test_page_outside_the_pool_gives_nan_for_its_sequence_only():
    B, Hq, Hkv, T, D, lens = 3, 4, 2, 3, 64, [100, 100, 100]
    inputs = make(B, Hq, Hkv, T, lens, D, BF16, 32, seed=9)
    want = oracle.decode_tree(*inputs[:5], lens, None, inputs[5], lam_of(Hq, BF16), D ** -0.5)
    for entry in (-1, inputs[3].shape[0], 1 << 30, -(1 << 31)):
        table = inputs[5].clone()
        table[1, 1] = entry
        o, lse = run(*inputs[:5], table, lens, None)
        assert torch.isnan(o[1]).all() and torch.isnan(lse[1]).all(), entry
        check((o[::2], lse[::2]), tuple(x[::2] for x in want), BF16)


def test_one_token_is_the_decode():
    """T = 1 over a contiguous cache against co_alibi_decode with the token appended, at split-K lengths."""
    for B, Hq, Hkv, L, D, dtype in [(1, 32, 8, 8192, 128, BF16), (2, 12, 12, 3001, 64, F16), (1, 8, 2, 70000, 128, F16),
                                    (1, 4, 2, 2500, 64, F32)]:
        gen = torch.Generator(device=DEV).manual_seed(L)
        n = lambda *s: (torch.randn(*s, generator=gen, device=DEV) * 0.5).to(dtype)  # noqa: B023,E731
        q, kc, vc = n(B, Hq, 1, D), n(B, Hkv, L + 1, D), n(B, Hkv, L + 1, D)
        k, v = kc[:, :, L:].clone(), vc[:, :, L:].clone()
        o, lse = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=L, return_lse=True)
        ro, rlse = co_alibi_decode(q, kc, vc, return_lse=True)
        eps = torch.finfo(dtype).eps
        # Each side rounds its weights and its output by half a step.
        assert (o.float() - ro.float()).abs().max() <= 2 * eps * vc.float().abs().max()
        assert (lse - rlse).abs().max() <= 1e-4 + 2e-6 * rlse.abs().max()


def test_chain_is_the_causal_attention():
    """A prompt in steps of up to 64 tokens over a growing paged cache gives co_alibi_attention's rows."""
    B, Hq, Hkv, S, D, page = 2, 8, 2, 333, 64, 32
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(B, S, H, D, generator=gen, device=DEV).to(F16).transpose(1, 2) for H in (Hq, Hkv, Hkv))
    want = co_alibi_attention(q, k, v, causal=True)
    blocks = -(-S // page)
    kc = torch.full((B * blocks, Hkv, page, D), math.nan, device=DEV, dtype=F16)
    vc = kc.clone()
    table = torch.randperm(B * blocks, generator=torch.Generator().manual_seed(2)).view(B, blocks).to(DEV, torch.int32)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    at = 0
    for T in (64, 1, 33, 64, 7, 64, 2, 64, 34):
        cut = slice(at, at + T)
        o = co_alibi_decode_tree(q[:, :, cut], k[:, :, cut], v[:, :, cut], kc, vc, seq_len=lens, block_table=table)
        # Both round their weights and their outputs to fp16: |v| <= 5.
        assert (o.float() - want[:, :, cut].float()).abs().max() <= 2 * torch.finfo(F16).eps * 5
        co_alibi_cache_append(k[:, :, cut], v[:, :, cut], kc, vc, lens, block_table=table)
        lens += T
        at += T
    assert at == S


def test_layouts_give_the_same_bits():
    """Strided new tokens, a (page, row, head, D) pool's transposed view, a layer of a larger pool, int64 indices."""
    B, Hq, Hkv, T, D, page, lens = 2, 8, 2, 9, 64, 16, [75, 130]
    q, k, v, kc, vc, table = (t.to(DEV) for t in make(B, Hq, Hkv, T, lens, D, BF16, page, seed=3))
    par = random_parents(B, T, torch.Generator().manual_seed(4)).to(DEV)
    lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par, block_table=table)

    def bshd(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    packed = torch.cat([bshd(x).transpose(1, 2).reshape(B, T, -1) for x in (q, k, v)], 2)
    pq, pk, pv = (x.view(B, T, -1, D).transpose(1, 2) for x in packed.split([Hq * D, Hkv * D, Hkv * D], 2))
    layers = torch.stack([torch.zeros_like(kc), kc, vc])
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=BF16)[1:].view(q.shape).copy_(q)  # not 16-byte aligned
    for label, args in [("strided", (bshd(q), bshd(k), bshd(v), kc, vc)), ("packed", (pq, pk, pv, kc, vc)),
                        ("pool", (q, k, v, bshd(kc), bshd(vc))), ("mixed", (q, k, v, kc, bshd(vc))),
                        ("layer", (q, k, v, layers[1], layers[2])), ("unaligned", (odd, k, v, kc, vc))]:
        got = co_alibi_decode_tree(*args, seq_len=lens, parents=par, block_table=table)
        assert torch.equal(got, want), label
    got = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens.long(), parents=par.long(), block_table=table.long())
    assert torch.equal(got, want)
    # One tree for every sequence; int64 values that would wrap into the valid range stay out of it.
    one = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par[0], block_table=table)
    assert torch.equal(one, co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par[:1].expand(B, T), block_table=table))
    wild = par.long().clone()
    wild[:, 3] = (1 << 32) + 1
    assert not co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=wild, block_table=table)[:, :, 3].any()


def test_lengths_are_clamped_and_bounded():
    B, Hq, Hkv, T, D = 3, 4, 2, 2, 64
    q, k, v, kc, vc, _ = (t if t is None else t.to(DEV) for t in make(B, Hq, Hkv, T, [64, 64, 64], D, F16, 0, seed=6))
    kc, vc = kc[:, :, :64].contiguous(), vc[:, :, :64].contiguous()
    got = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=torch.tensor([-5, 1 << 30, 40], device=DEV), max_seq_len=50)
    want = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=torch.tensor([0, 50, 40], device=DEV), max_seq_len=50)
    assert torch.equal(got, want)
    nothing = co_alibi_decode_tree(q, k, v, kc[:, :, :0], vc[:, :, :0])
    assert torch.equal(nothing, co_alibi_decode_tree(q, k, v, kc, vc, seq_len=0))
    assert co_alibi_decode_tree(q[:, :, :0], k[:, :, :0], v[:, :, :0], kc, vc).shape == (B, Hq, 0, D)
    assert co_alibi_decode_tree(q[:0], k[:0], v[:0], kc[:0], vc[:0]).shape == (0, Hq, T, D)


def test_cache_past_32_bit_offsets():
    """Pages whose element offsets pass 2^32 (one pool of 9 GB serves as K and V)."""
    Hkv, page, D, T, L = 8, 256, 128, 5, 700
    pages = (1 << 32) // (Hkv * page * D) + 64
    pool = torch.empty(pages, Hkv, page, D, device=DEV, dtype=F16)
    gen = torch.Generator(device=DEV).manual_seed(8)
    n = lambda *s: (torch.randn(*s, generator=gen, device=DEV) * 0.5).to(F16)  # noqa: E731
    far = [pages - 1, 3, pages - 40]
    small = n(3, Hkv, page, D)
    for i, p in enumerate(far):
        pool[p] = small[i]
    q, k, v = n(1, 16, T, D), n(1, Hkv, T, D), n(1, Hkv, T, D)
    got = co_alibi_decode_tree(q, k, v, pool, pool, seq_len=L, block_table=torch.tensor([far], dtype=torch.int32, device=DEV))
    near = co_alibi_decode_tree(q, k, v, small, small, seq_len=L,
                                block_table=torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV))
    assert torch.equal(got, near)


def test_refusals_on_the_device():
    q, k, v, kc, vc, table = (t.to(DEV) for t in make(2, 4, 2, 3, [20, 20], 64, F16, 16))
    for kw, err, msg in [
            (dict(k_cache=kc[:, :, :, ::2].repeat(1, 1, 1, 2).transpose(2, 3).contiguous().transpose(2, 3)), ValueError, "dense"),
            (dict(k_cache=kc[:, :1], v_cache=vc[:, :1]), ValueError, "k's heads and head dim"),
            (dict(v_cache=vc[:-1]), ValueError, "of one shape"),
            (dict(k_cache=kc[:, :, :8], v_cache=vc[:, :, :8]), ValueError, "power of two"),
            (dict(block_table=None), ValueError, "one entry per sequence"),
            (dict(block_table=table.float()), TypeError, "int32 or int64"),
            (dict(parents=torch.zeros(2, 4, dtype=torch.int32, device=DEV)), ValueError, "parents must be"),
            (dict(parents=torch.zeros(3, device=DEV)), TypeError, "int32 or int64"),
            (dict(k_cache=kc.bfloat16()), TypeError, "share one dtype"),
    ]:
        args = dict(k_cache=kc, v_cache=vc, block_table=table, seq_len=10)
        args.update(kw)
        with pytest.raises(err, match=msg):
            co_alibi_decode_tree(q, k, v, **args)


def test_capture_and_other_streams():
    B, Hq, Hkv, T, D, page = 2, 8, 2, 6, 128, 64
    q, k, v, kc, vc, table = (t.to(DEV) for t in make(B, Hq, Hkv, T, [2000, 900], D, BF16, page, seed=12))
    lens = torch.tensor([2000, 900], dtype=torch.int32, device=DEV)
    par = random_parents(B, T, torch.Generator().manual_seed(1)).to(DEV)
    want = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par, block_table=table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par, block_table=table)
    side.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par, block_table=table)
    for i in range(4):
        lens.copy_(torch.tensor([2000 - 300 * i, 900 - i], dtype=torch.int32))
        q.mul_(-0.7)
        graph.replay()
        torch.cuda.synchronize()
        eager = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, parents=par, block_table=table)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_slopes_of_other_bias_max():
    inputs = make(1, 6, 2, 4, [90], 64, F32, 16, seed=2)
    for bias_max in (0.0, 4.0, 16.0):
        want = oracle.decode_tree(*inputs[:5], [90], None, inputs[5], lam_of(6, F32, bias_max), 0.2)
        check(run(*inputs, [90], None, bias_max=bias_max, sm_scale=0.2), want, F32)
