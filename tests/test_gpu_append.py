"""co_alibi_cache_append: a copy, so every byte of the caches is compared.  Needs an MI355X."""
import pytest
import torch

from co_alibi_attn import co_alibi_cache_append
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


def make(B, Hkv, T, D, dtype, page, capacity, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    k, v = n(B, Hkv, T, D), n(B, Hkv, T, D)
    if page == 0:
        return k, v, n(B, Hkv, capacity, D), n(B, Hkv, capacity, D), None
    blocks = -(-capacity // page)
    table = torch.randperm(B * blocks + 1, generator=gen)[:B * blocks].view(B, blocks).to(torch.int32)
    return k, v, n(B * blocks + 1, Hkv, page, D), n(B * blocks + 1, Hkv, page, D), table


def run_and_check(k, v, kc, vc, table, lens, rows=None, counts=None):
    want = oracle.cache_append(k, v, kc, vc, lens, table, rows, counts)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    dk, dv = kc.to(DEV), vc.to(DEV)
    out = co_alibi_cache_append(dev(k), dev(v), dk, dv, dev(lens), block_table=dev(table), rows=dev(rows), counts=dev(counts))
    torch.cuda.synchronize()
    assert out is None and same(dk, want[0]) and same(dv, want[1])


@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
@pytest.mark.parametrize("case", [
    # B, Hkv, T, D, page, capacity
    (1, 1, 1, 16, 0, 5), (3, 2, 1, 64, 16, 100), (2, 12, 7, 64, 0, 40), (2, 8, 33, 128, 16, 90), (1, 3, 300, 256, 64, 400),
    (5, 1, 2, 32, 256, 300),
], ids=str)
def test_append_matches_oracle(case, dtype):
    B, Hkv, T, D, page, cap = case
    gen = torch.Generator().manual_seed(T)
    k, v, kc, vc, table = make(*case[:4], dtype, page, cap, seed=D)
    room = kc.shape[2] if page == 0 else page * table.shape[1]
    lens = torch.randint(0, room - T + 1, (B,), generator=gen, dtype=torch.int32)
    run_and_check(k, v, kc, vc, table, lens)
    run_and_check(k, v, kc, vc, table, lens, counts=torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32))
    n = min(T, 5)
    rows = torch.randint(0, T, (B, n), generator=gen, dtype=torch.int32)  # the same row more than once
    run_and_check(k, v, kc, vc, table, lens, rows=rows)
    run_and_check(k, v, kc, vc, table, lens, rows=rows, counts=torch.randint(0, n + 1, (B,), generator=gen, dtype=torch.int32))


def test_more_rows_than_new_tokens():
    k, v, kc, vc, table = make(2, 2, 2, 64, F16, 16, 64)
    rows = torch.tensor([[1, 0, 1, 1, 0, 1, 0], [0, 0, 0, 1, 1, 1, 0]], dtype=torch.int32)
    run_and_check(k, v, kc, vc, table, torch.tensor([0, 50], dtype=torch.int32), rows=rows)


@pytest.mark.parametrize("page", (0, 16))
def test_rows_without_a_place_are_left_out(page):
    k, v, kc, vc, table = make(4, 2, 6, 64, BF16, page, 32, seed=1)
    lens = torch.tensor([30, -3, 1 << 30, 5], dtype=torch.int32)
    run_and_check(k, v, kc, vc, table, lens)
    run_and_check(k, v, kc, vc, table, lens, counts=torch.tensor([9, 5, -1, 1 << 30], dtype=torch.int32))
    rows = torch.tensor([[0, -1, 6, 5], [1, 2, 3, 4], [0, 0, 0, 0], [1 << 30, 2, -(1 << 31), 3]], dtype=torch.int32)
    run_and_check(k, v, kc, vc, table, lens.clamp(max=20), rows=rows)
    if page:
        for entry in (-1, kc.shape[0], 1 << 30):
            bad = table.clone()
            bad[3, 0] = entry
            run_and_check(k, v, kc, vc, bad, lens)


def test_layouts():
    """Transposed and packed sources, an unaligned one, a (page, row, head, D) pool, int64 indices."""
    B, Hkv, T, D, page = 2, 3, 9, 64, 16
    k, v, kc, vc, table = make(B, Hkv, T, D, F16, page, 60, seed=2)
    lens = torch.tensor([3, 40], dtype=torch.int32)
    want = oracle.cache_append(k, v, kc, vc, lens, table, None, None)
    bshd = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    packed = torch.stack([k.transpose(1, 2), v.transpose(1, 2)], 2).to(DEV)
    pk, pv = packed[:, :, 0].transpose(1, 2), packed[:, :, 1].transpose(1, 2)
    odd = torch.empty(k.numel() + 1, dtype=F16, device=DEV)[1:].view(k.shape).copy_(k)
    for label, nk, nv, wrap in [("strided", bshd(k.to(DEV)), v.to(DEV), lambda t: t), ("packed", pk, pv, lambda t: t),
                                ("unaligned", odd, v.to(DEV), lambda t: t), ("pool", k.to(DEV), v.to(DEV), bshd)]:
        dk, dv = wrap(kc.to(DEV)), wrap(vc.to(DEV))
        co_alibi_cache_append(nk, nv, dk, dv, lens.to(DEV), block_table=table.to(DEV))
        assert same(dk.contiguous(), want[0]) and same(dv.contiguous(), want[1]), label
    dk, dv = kc.to(DEV), vc.to(DEV)
    before = dk._version
    co_alibi_cache_append(k.to(DEV), v.to(DEV), dk, dv, lens.to(DEV).long(), block_table=table.to(DEV).long())
    assert same(dk, want[0]) and same(dv, want[1]) and dk._version > before


def test_empty_calls_write_nothing():
    k, v, kc, vc, table = (t.to(DEV) for t in make(2, 2, 3, 64, F16, 16, 32))
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    keep = kc.clone()
    co_alibi_cache_append(k[:, :, :0], v[:, :, :0], kc, vc, lens, block_table=table)
    co_alibi_cache_append(k, v, kc, vc, lens, block_table=table, rows=torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    co_alibi_cache_append(k[:0], v[:0], kc, vc, lens[:0], block_table=table[:0])
    assert same(kc, keep)


def test_refusals_on_the_device():
    k, v, kc, vc, table = (t.to(DEV) for t in make(2, 2, 3, 64, F16, 16, 32))
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    for args, kw, err, msg in [
            ((k, v, kc, vc, lens[:1]), {}, ValueError, "seq_lens must be"),
            ((k, v, kc, vc, lens.float()), {}, TypeError, "int32 or int64"),
            ((k, v, kc, vc, lens), dict(counts=lens[:1]), ValueError, "counts must be"),
            ((k, v, kc, vc, lens), dict(rows=lens), ValueError, "rows must be"),
            ((k, v, kc[:1].expand(5, -1, -1, -1), vc[:1].expand(5, -1, -1, -1), lens), {}, RuntimeError, "overlap"),
            ((k, v, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, lens), {}, ValueError, "dense"),
    ]:
        with pytest.raises(err, match=msg):
            co_alibi_cache_append(*args, block_table=table, **kw)


def test_capture():
    k, v, kc, vc, table = (t.to(DEV) for t in make(2, 2, 1, 64, F16, 16, 64))
    lens = torch.tensor([0, 7], dtype=torch.int32, device=DEV)
    co_alibi_cache_append(k, v, kc, vc, lens, block_table=table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        co_alibi_cache_append(k, v, kc, vc, lens, block_table=table)
    want = [kc.cpu(), vc.cpu()]
    for i in range(5):
        k.add_(1.0)
        v.mul_(-2.0)
        lens.add_(3)
        graph.replay()
        torch.cuda.synchronize()
        want = oracle.cache_append(k.cpu(), v.cpu(), *want, lens.cpu(), table.cpu(), None, None)
        assert same(kc, want[0]) and same(vc, want[1]), i


def test_offsets_past_32_bits():
    """A pool whose element offsets pass 2^32 (9 GB), as keys; the values' pool is a small one of the same shape
    of page, so a second call writes the same pages through the value operand."""
    Hkv, page, D, T = 8, 256, 128, 5
    pages = (1 << 32) // (Hkv * page * D) + 8
    pool = torch.zeros(pages, Hkv, page, D, device=DEV, dtype=F16)
    k = torch.randn(1, Hkv, T, D, device=DEV).to(F16)
    v = torch.randn(1, Hkv, T, D, device=DEV).to(F16)
    table = torch.tensor([[pages - 1, 2, pages - 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([2 * page - 2], dtype=torch.int32, device=DEV)  # two rows in page 2, three in pages - 3
    other = torch.zeros_like(pool)
    co_alibi_cache_append(k, v, pool, other, lens, block_table=table)
    for cache, new in ((pool, k), (other, v)):
        assert torch.equal(cache[2, :, -2:], new[0, :, :2]) and torch.equal(cache[pages - 3, :, :3], new[0, :, 2:])
        assert int(torch.count_nonzero(cache[2])) + int(torch.count_nonzero(cache[pages - 3])) == int(torch.count_nonzero(new))
        assert not cache[3:pages - 3].any() and not cache[:2].any() and not cache[pages - 2:].any()
