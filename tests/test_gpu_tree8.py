"""co_alibi_decode_tree_8bit against the float64 oracle (oracle/serving8.py).  Needs an MI355X.

Tolerances: the oracle's first-order bound of what fp32 arithmetic and the rounding of the weights to the input type can
change, plus half a step of the output type.
"""
import math

import pytest
import torch

from co_alibi_attn import (_native, co_alibi_cache_append_8bit, co_alibi_cache_read_8bit, co_alibi_decode_tree,
                           co_alibi_decode_tree_8bit)
from oracle import co_alibi_ref as ref
from oracle import serving8 as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
NAME = {F16: "fp16", BF16: "bf16", F32: "fp32"}
FORMATS = pytest.mark.parametrize("fmt", (E4M3, INT8), ids=("e4m3", "int8"))


def random_parents(B, T, gen, absent=False):
    par = torch.stack([torch.arange(T) - torch.randint(1, 6, (T,), generator=gen) for _ in range(B)]).clamp_(min=-1)
    if absent:  # a node of its own as parent, a later one, one below -1: each takes its descendants with it
        for b in range(B):
            for bad in (lambda t: t, lambda t: t + 1, lambda t: -2, lambda t: 1 << 30):
                t = int(torch.randint(0, T, (1,), generator=gen))
                par[b, t] = bad(t)
    return par.to(torch.int32)


def quantise(x, fmt):
    """Codes and scales of (units, Hkv, rows, D), from a power of two for every block of 16 rows."""
    U, H, n, D = x.shape
    blocks = -(-n // 16)
    y = torch.nn.functional.pad(x, (0, 0, 0, blocks * 16 - n)).view(U, H, blocks, 16, D).double()
    s = torch.exp2(torch.ceil(torch.log2(y.abs().amax((3, 4)) / oracle.LARGEST[fmt])).clamp(min=-40))
    c = oracle.code(y / s[..., None, None], fmt).view(U, H, blocks * 16, D)[:, :, :n]
    return c.to(fmt), s.float()


def make(B, Hq, Hkv, T, lens, D, dtype, fmt, page, seed=0, scale=0.5, spread=1.0):
    """Inputs on the CPU.  Rows that no sequence has filled, pages that none uses and their scales hold garbage: the codes of
    NaN where the format has any, scales of NaN."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen) * scale  # noqa: E731
    q, k, v = n(B, Hq, T, D).to(dtype), n(B, Hkv, T, D).to(dtype), n(B, Hkv, T, D).to(dtype)
    rows = max(max(lens), 1)
    blocks = -(-rows // page) if page else 0
    units, per = (B * blocks + 2, page) if page else (B, rows + 3)
    table = torch.randperm(units, generator=gen)[:B * blocks].view(B, blocks).to(torch.int32) if page else None
    size = torch.exp2(spread * torch.randn(2, units, Hkv, -(-per // 16), generator=gen)).repeat_interleave(16, 3)[..., :per, None]
    caches, scales = zip(*(quantise(n(units, Hkv, per, D) * size[i], fmt) for i in range(2)))
    used = torch.zeros(units, -(-per // 16) * 16, dtype=torch.bool)
    for b in range(B):
        for r in range(lens[b]):
            used[(int(table[b, r // page]), r % page) if page else (b, r)] = True
        if page:
            table[b, -(-lens[b] // page):] = -7  # entries past the filled rows are never read
    for c, s in zip(caches, scales):
        c.view(torch.uint8).masked_fill_(~used[:, None, :per, None], 0x7f)
        s.masked_fill_(~used.view(units, -1, 16).any(2)[:, None], math.nan)
    return q, k, v, caches, scales, table


def dev(t):
    return None if t is None else t.to(DEV)


def run(q, k, v, caches, scales, table, lens, parents, **kw):
    o, lse = co_alibi_decode_tree_8bit(dev(q), dev(k), dev(v), *map(dev, caches), *map(dev, scales), parents=dev(parents),
                                       block_table=dev(table), seq_len=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                       return_lse=True, **kw)
    torch.cuda.synchronize()
    return o.cpu(), lse.cpu()


def within(o, lse, want):
    """Inside the oracle's bounds; o has been rounded once more."""
    ro, rlse, ob, lb = want
    half = torch.finfo(o.dtype).eps / 2
    tiny = torch.finfo(F16).tiny * half if o.dtype == F16 else 0.0  # fp16 steps are 2^-24 below its normals
    assert torch.isfinite(o).all()
    over = (o.double() - ro).abs() - (half * (ro.abs() + ob) + ob + tiny)
    assert over.max() <= 0, f"o off by {over.max():.2e} beyond its bound"
    dead = rlse == -math.inf
    assert torch.equal(lse == -math.inf, dead) and (o[dead] == 0).all()
    over = torch.where(dead, 0.0, (lse.double() - rlse).abs() - lb)
    assert over.max() <= 0, f"lse off by {over.max():.2e} beyond its bound"


def check(q, k, v, caches, scales, table, lens, parents, o, lse, bias_max=8.0, sm_scale=None):
    full = parents if parents is None or parents.dim() == 2 else parents.expand(q.shape[0], -1)
    within(o, lse, oracle.decode_tree(q, k, v, caches, scales, lens, full, table, slopes(q.shape[1], bias_max, q.dtype),
                                      q.shape[3] ** -0.5 if sm_scale is None else sm_scale))


def slopes(heads, bias_max, dtype):
    return ref.slopes(heads, bias_max, dtype=dtype).float()


@FORMATS
@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
@pytest.mark.parametrize("case", [
    # B, Hq, Hkv, T, lens, D, page
    (1, 1, 1, 1, [1], 16, 0), (2, 4, 4, 1, [33, 500], 64, 16), (3, 12, 12, 1, [0, 17, 300], 64, 64), (2, 8, 2, 3, [100, 129], 128, 0),
    (1, 8, 1, 7, [700], 32, 32), (4, 8, 2, 16, [5, 0, 160, 1000], 128, 16), (2, 4, 1, 64, [31, 260], 64, 256),
    (1, 6, 2, 33, [90], 16, 16), (1, 2, 1, 40, [65], 256, 64), (2, 16, 1, 2, [16, 15], 128, 16),
], ids=str)
def test_matches_oracle(case, dtype, fmt):
    B, Hq, Hkv, T, lens, D, page = case
    if dtype == F32 and D == 256:
        pytest.skip("head dim 256 needs fp16 or bf16")
    gen = torch.Generator().manual_seed(T)
    args = make(B, Hq, Hkv, T, lens, D, dtype, fmt, page, seed=D + T)
    for parents in (None, random_parents(B, T, gen), random_parents(B, T, gen, absent=True)):
        check(*args, lens, parents, *run(*args, lens, parents))


@FORMATS
@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
def test_long_and_ragged(dtype, fmt):
    """Splits and their merge, also under a plan of their own lengths."""
    for B, Hq, Hkv, T, lens, D, page in ((1, 4, 1, 5, [9001], 64, 64), (6, 4, 2, 1, [7000, 3, 0, 2500, 6999, 16], 32, 16)):
        args = make(B, Hq, Hkv, T, lens, D, dtype, fmt, page, seed=B)
        check(*args, lens, None, *run(*args, lens, None))


@FORMATS
@pytest.mark.parametrize("spread", (0.0, 4.0))
def test_scales_of_very_different_size(spread, fmt):
    """Blocks of V 2^30 apart from one another, and blocks of zeros, whose scale is the smallest."""
    for dtype in (BF16, F32):
        lens = [333, 64]
        q, k, v, caches, scales, table = make(2, 4, 2, 5, lens, 64, dtype, fmt, 16, seed=9, spread=spread)
        scales = [s.clone() for s in scales]
        scales[1][:, :, 0] *= torch.exp2(torch.arange(scales[1].shape[0]) % 31 - 15.0)[:, None]
        zero = int(table[0, 3])
        caches[1].view(torch.uint8)[zero] = 0
        scales[1][zero] = 2.0 ** -40
        scales[0][int(table[1, 1])] *= 1.37  # no power of two
        args = q, k, v, caches, scales, table
        check(*args, lens, None, *run(*args, lens, None))


@FORMATS
def test_bad_pages_and_scales_make_their_sequence_nan(fmt):
    lens = [200, 170, 40, 90]
    q, k, v, caches, scales, table = make(4, 4, 2, 3, lens, 64, BF16, fmt, 16, seed=4)
    want, want_lse = run(q, k, v, caches, scales, table, lens, None)
    assert torch.isfinite(want).all()
    for entry in (-1, caches[0].shape[0], 1 << 30):
        bad = table.clone()
        bad[1, 5] = entry
        o, lse = run(q, k, v, caches, scales, bad, lens, None)
        assert torch.isnan(o[1]).all() and torch.isnan(lse[1]).all()
        keep = [0, 2, 3]
        assert torch.equal(o[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])
    for i in range(2):
        for x in (math.nan, 0.0, -1.0, math.inf, 2.0 ** -41, 2.0 ** 41):
            bad = [s.clone() for s in scales]
            bad[i][int(table[3, 5]), 1, 0] = x  # rows 80 to 90, kv head 1
            o, lse = run(q, k, v, caches, bad, table, lens, None)
            assert torch.isnan(o[3, 2:]).all() and torch.isnan(lse[3, 2:]).all()
            assert torch.equal(o[:3], want[:3]) and torch.equal(o[3, :2], want[3, :2])


@FORMATS
def test_values_of_tokens_that_are_not_seen(fmt):
    """An infinity or a NaN of a new token reaches the tokens that see it, and no other."""
    lens = [50]
    for T in (6, 40):
        q, k, v, caches, scales, table = make(1, 4, 2, T, lens, 64, BF16, fmt, 16, seed=T)
        parents = torch.arange(-1, T - 1, dtype=torch.int32)
        parents[3:] = 0  # tokens 1 -> 2, and the others, hang on token 0
        want, want_lse = run(q, k, v, caches, scales, table, lens, parents)
        k2, v2 = k.clone(), v.clone()
        v2[0, 0, 2, 7], v2[0, 1, 2, 9] = math.inf, math.nan
        k2[0, 0, T - 1, 3] = math.nan
        o, lse = run(q, k2, v2, caches, scales, table, lens, parents)
        others = [t for t in range(T) if t not in (2, T - 1)]
        assert torch.equal(o[:, :, others], want[:, :, others]) and torch.equal(lse[:, :, others], want_lse[:, :, others])
        assert (o[0, :2, 2, 7] == math.inf).all() and torch.isnan(o[0, 2:, 2, 9]).all()
        assert torch.isfinite(o[0, :2, 2, :7]).all() and torch.isnan(o[0, :2, T - 1]).all()
        assert torch.equal(o[0, 2:, T - 1], want[0, 2:, T - 1])


@FORMATS
def test_agrees_with_the_decode_over_values(fmt):
    """Over the values that the cache holds, read back (exact in fp32), co_alibi_decode_tree gives the same up to fp32's bound."""
    lens = [300, 77]
    args = make(2, 8, 2, 9, lens, 64, F32, fmt, 16, seed=6)
    q, k, v, caches, scales, table = args
    o, lse = run(*args, lens, None)
    check(*args, lens, None, o, lse)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kc, vc = co_alibi_cache_read_8bit(*map(dev, caches), *map(dev, scales), seq, 300, dtype=F32, block_table=dev(table))
    o2, lse2 = co_alibi_decode_tree(dev(q), dev(k), dev(v), kc, vc, seq_len=seq, return_lse=True)
    check(*args, lens, None, o2.cpu(), lse2.cpu())


def test_lengths_strides_and_settings():
    """Clamped lengths, one length for all, a bound, packed projections, int64 tables, another scale and bias_max."""
    lens = [300, 77]
    args = make(2, 4, 2, 5, lens, 128, BF16, E4M3, 16, seed=8)
    q, k, v, caches, scales, table = args
    o, lse = run(*args, lens, None)
    check(*args, lens, None, o, lse)
    packed = torch.cat([x.transpose(1, 2) for x in (q, k, v)], 2).to(DEV)  # (B, T, Hq + 2 Hkv, D)
    pq, pk, pv = (x.transpose(1, 2) for x in packed.split((4, 2, 2), 2))
    c, s = [dev(t) for t in caches], [dev(t) for t in scales]
    o2 = co_alibi_decode_tree_8bit(pq, pk, pv, *c, *s, seq_len=torch.tensor(lens, device=DEV), block_table=table.to(DEV).long())
    assert torch.equal(o2.cpu(), o)
    wide = [torch.stack([t.view(torch.uint8)] * 2, 1)[:, 1].view(E4M3) for t in c]
    wide_s = [torch.stack([t] * 2, 1)[:, 1] for t in s]
    o2 = co_alibi_decode_tree_8bit(pq, pk, pv, *wide, *wide_s, seq_len=torch.tensor(lens, device=DEV), block_table=dev(table))
    assert torch.equal(o2.cpu(), o)
    high = torch.tensor([1 << 30, -5], dtype=torch.int32, device=DEV)
    table2 = table.clone()
    table2[1] = table2[0]
    o3, l3 = co_alibi_decode_tree_8bit(dev(q), dev(k), dev(v), *c, *s, seq_len=high, block_table=dev(table2), max_seq_len=300,
                                       return_lse=True)
    check(q, k, v, caches, scales, table2, [300, 0], None, o3.cpu(), l3.cpu())
    o3, l3 = co_alibi_decode_tree_8bit(dev(q), dev(k), dev(v), *c, *s, seq_len=70, block_table=dev(table), return_lse=True,
                                       sm_scale=0.2, bias_max=4.0)
    check(q, k, v, caches, scales, table, [70, 70], None, o3.cpu(), l3.cpu(), bias_max=4.0, sm_scale=0.2)


def test_tail_skip():
    """With the tail skip or without it, a long steep sequence is within the bound."""
    lens = [4000]
    args = make(1, 8, 2, 24, lens, 64, BF16, E4M3, 64, seed=10)
    for skip in (True, False):
        with _native.tail_skip(skip):
            check(*args, lens, None, *run(*args, lens, None))


def test_a_step_captured_and_replayed():
    """Append, decode and lengths in one graph, replayed over a growing cache; a second graph and a side stream beside it."""
    B, Hq, Hkv, D, page, cap = 2, 4, 2, 64, 16, 96
    gen = torch.Generator().manual_seed(2)
    new = [torch.randn(B, h, 60, D, generator=gen).to(BF16) for h in (Hq, Hkv, Hkv)]
    blocks = cap // page
    table = torch.randperm(B * blocks, generator=gen).view(B, blocks).to(torch.int32)
    caches = [torch.zeros(B * blocks, Hkv, page, D, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(B * blocks, Hkv, 1, device=DEV) for _ in range(2)]
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(B, x.shape[1], 1, D, dtype=BF16, device=DEV) for x in new)
    tab = table.to(DEV)

    def step():
        o = co_alibi_decode_tree_8bit(q, k, v, *caches, *scales, seq_len=lens, block_table=tab)
        co_alibi_cache_append_8bit(k, v, *caches, *scales, lens, block_table=tab)
        lens.add_(1)
        return o

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lens.zero_()
    host_c = [torch.zeros(B * blocks, Hkv, page, D, dtype=torch.int8) for _ in range(2)]
    host_s = [torch.zeros(B * blocks, Hkv, 1) for _ in range(2)]
    for i in range(50):
        for dst, src in zip((q, k, v), new):
            dst.copy_(src[:, :, i:i + 1])
        # (Before the append, which may round the cache's last block again.)
        eager = co_alibi_decode_tree_8bit(q, k, v, *caches, *scales, seq_len=lens, block_table=tab)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, out)
        nq, nk, nv = (x[:, :, i:i + 1] for x in new)
        if i % 7 == 0:
            want, _, ob, _ = oracle.decode_tree(nq, nk, nv, host_c, host_s, [i] * B, None, table, slopes(Hq, 8.0, BF16), D ** -0.5)
            assert ((out.cpu().double() - want).abs() <= ob * 1.01 + 2.0 ** -8 * want.abs()).all()
        host_c, host_s = oracle.append(nk, nv, host_c, host_s, [i] * B, table, None, None)


def test_two_streams_at_once():
    lens = [2000, 1500]
    many = [make(2, 8, 2, 4, lens, 64, F16, E4M3, 64, seed=s) for s in (1, 2)]
    want = [run(*a, lens, None)[0] for a in many]
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    on = [([dev(x) for x in a[:3]], [dev(x) for x in a[3]], [dev(x) for x in a[4]], dev(a[5])) for a in many]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in many]
    got = [[], []]
    for _ in range(10):
        for i, ((q, k, v), c, s, t) in enumerate(on):
            with torch.cuda.stream(streams[i]):
                got[i].append(co_alibi_decode_tree_8bit(q, k, v, *c, *s, seq_len=seq, block_table=t))
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for g, w in zip(got, want) for o in g)


def test_rows_past_32_bits():
    """A pool of more than 2^32 bytes, the sequence's pages at both of its ends."""
    Hkv, D, page = 8, 128, 64
    pages = (1 << 32) // (Hkv * D * page) + 5
    small = make(1, 8, Hkv, 2, [150], D, BF16, INT8, page, seed=1)
    q, k, v, caches, scales, table = small
    where = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    big_c = [torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=DEV) for _ in range(2)]
    big_s = [torch.full((pages, Hkv, page // 16), math.nan, device=DEV) for _ in range(2)]
    for j in range(3):
        for x, y in zip((*big_c, *big_s), (*caches, *scales)):
            x[int(where[0, j])] = y[int(table[0, j])].to(DEV)
    o, lse = run(*small, [150], None)
    o2 = co_alibi_decode_tree_8bit(dev(q), dev(k), dev(v), *big_c, *big_s, seq_len=150, block_table=dev(where))
    check(*small, [150], None, o, lse)
    assert torch.equal(o2.cpu(), o)


def test_empty_calls():
    q, k, v, caches, scales, table = make(2, 4, 2, 3, [5, 9], 64, BF16, E4M3, 16)
    c, s = [dev(t) for t in caches], [dev(t) for t in scales]
    o, lse = co_alibi_decode_tree_8bit(dev(q)[:, :, :0], dev(k)[:, :, :0], dev(v)[:, :, :0], *c, *s, seq_len=0,
                                       block_table=dev(table), return_lse=True)
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    o, lse = co_alibi_decode_tree_8bit(dev(q), dev(k), dev(v), *c, *s, seq_len=0, block_table=dev(table)[:, :0], return_lse=True)
    check(q, k, v, caches, scales, table, [0, 0], None, o.cpu(), lse.cpu())
