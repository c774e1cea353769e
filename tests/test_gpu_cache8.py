"""co_alibi_cache_append_8bit and co_alibi_cache_read_8bit against the float64 oracle (oracle/serving8.py): codes and scales are
whole numbers and powers of two, so every byte is compared.  Needs an MI355X."""
import math

import pytest
import torch

from co_alibi_attn import co_alibi_cache_append_8bit, co_alibi_cache_read_8bit
from oracle import serving8 as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
FORMATS = pytest.mark.parametrize("fmt", (E4M3, INT8), ids=("e4m3", "int8"))


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


def same_scales(a, b):
    return torch.equal(torch.nan_to_num(a.cpu(), nan=-1.0), torch.nan_to_num(b.cpu(), nan=-1.0))


def codes(gen, shape, fmt):
    """Random codes, none of them a NaN."""
    if fmt == INT8:
        return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8)
    x = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8)
    return torch.where((x & 127) == 127, 5, x).to(torch.uint8).view(fmt)


def make(B, Hkv, T, D, dtype, fmt, page, capacity, seed=0):
    """New keys and values whose rows differ in size, and a cache with random codes and scales."""
    gen = torch.Generator().manual_seed(seed)

    def new():
        x = torch.randn(B, Hkv, T, D, generator=gen) * torch.exp2(4 * torch.randn(B, Hkv, T, 1, generator=gen))
        return x.to(dtype)

    k, v = new(), new()
    blocks = -(-capacity // page) if page else 0
    units, rows = (B * blocks + 1, page) if page else (B, capacity)
    table = torch.randperm(units, generator=gen)[:B * blocks].view(B, blocks).to(torch.int32) if page else None
    caches = [codes(gen, (units, Hkv, rows, D), fmt) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, 3, (units, Hkv, -(-rows // 16)), generator=gen).float()) for _ in range(2)]
    return k, v, caches, scales, table


def dev(t):
    return None if t is None else t.to(DEV)


def run_and_check(k, v, caches, scales, table, lens, rows=None, counts=None):
    want, want_scales = oracle.append(k, v, caches, scales, lens, table, rows, counts)
    c, s = [dev(t) for t in caches], [dev(t) for t in scales]
    out = co_alibi_cache_append_8bit(dev(k), dev(v), *c, *s, dev(lens), block_table=dev(table), rows=dev(rows), counts=dev(counts))
    torch.cuda.synchronize()
    assert out is None
    for got, exp in zip(s, want_scales):
        assert same_scales(got, exp)
    for got, exp in zip(c, want):
        assert same(got, exp)
    return c, s


@FORMATS
@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
@pytest.mark.parametrize("case", [
    # B, Hkv, T, D, page, capacity
    (1, 1, 1, 16, 0, 5), (3, 2, 1, 64, 16, 100), (2, 3, 7, 64, 0, 41), (2, 2, 33, 128, 16, 90), (1, 2, 130, 256, 64, 200),
    (4, 1, 2, 32, 256, 300), (5, 2, 20, 16, 32, 64),
], ids=str)
def test_append_matches_oracle(case, dtype, fmt):
    B, Hkv, T, D, page, cap = case
    gen = torch.Generator().manual_seed(T)
    k, v, caches, scales, table = make(*case[:4], dtype, fmt, page, cap, seed=D)
    room = cap if page == 0 else page * table.shape[1]
    lens = torch.randint(0, room - T + 1, (B,), generator=gen, dtype=torch.int32)
    run_and_check(k, v, caches, scales, table, lens)
    run_and_check(k, v, caches, scales, table, lens // 16 * 16)
    run_and_check(k, v, caches, scales, table, lens, counts=torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32))
    n = min(T, 5)
    rows = torch.randint(0, T, (B, n), generator=gen, dtype=torch.int32)  # the same row more than once
    run_and_check(k, v, caches, scales, table, lens, rows=rows, counts=torch.randint(0, n + 1, (B,), generator=gen, dtype=torch.int32))


@FORMATS
@pytest.mark.parametrize("page", (0, 16))
def test_rows_without_a_place_are_left_out(page, fmt):
    k, v, caches, scales, table = make(4, 2, 6, 64, BF16, fmt, page, 32, seed=1)
    lens = torch.tensor([30, -3, 1 << 30, 5], dtype=torch.int32)
    run_and_check(k, v, caches, scales, table, lens)
    run_and_check(k, v, caches, scales, table, lens, counts=torch.tensor([9, 5, -1, 1 << 30], dtype=torch.int32))
    rows = torch.tensor([[0, -1, 6, 5], [1, 2, 3, 4], [0, 0, 0, 0], [1 << 30, 2, -(1 << 31), 3]], dtype=torch.int32)
    run_and_check(k, v, caches, scales, table, lens.clamp(max=20), rows=rows)
    run_and_check(k, v, caches, scales, table, lens.clamp(max=20), rows=torch.full((4, 3), -1, dtype=torch.int32))
    if page:
        for entry in (-1, caches[0].shape[0], 1 << 30):
            bad = table.clone()
            bad[3, 0] = entry
            run_and_check(k, v, caches, scales, bad, lens)


@FORMATS
def test_rounding_and_the_choice_of_a_scale(fmt):
    """Every bfloat16 near the borders of a power of two, ties, the largest codes and the smallest steps."""
    most = oracle.LARGEST[fmt]
    x = torch.cat([torch.arange(-most, most + 1, 0.5), torch.linspace(-most, most, 999), 2.0 ** torch.arange(-30, 9.0),
                   torch.tensor([most, -most, 0.0, -0.0])]).float()
    x = torch.nn.functional.pad(x, (0, -len(x) % 64)).view(1, 1, -1, 64)
    T = x.shape[2]
    for factor in (1.0, 0.5, 1.0001, 0.9999, 2.0 ** -30, 2.0 ** -50, 3.0e-39, 2.0 ** 30, 2.0 ** 40, 2.0 ** 41, 0.0):
        blank = [torch.zeros(1, 1, T, 64, dtype=torch.int8).view(fmt) for _ in range(2)]
        scales = [torch.zeros(1, 1, -(-T // 16)) for _ in range(2)]
        run_and_check(x * factor, -x * factor, blank, scales, None, torch.zeros(1, dtype=torch.int32))


@FORMATS
def test_a_growing_block_stays_within_one_step(fmt):
    """Sixteen single appends, each larger than the one before: every value within one step of the last scale's codes (e4m3:
    within 2^-4 of itself, or 2^-9 steps)."""
    gen = torch.Generator().manual_seed(3)
    k = torch.randn(1, 2, 16, 64, generator=gen) * torch.exp2(torch.arange(16.0) * 0.7)[:, None]
    caches = [torch.zeros(1, 2, 16, 64, dtype=torch.int8, device=DEV).view(fmt) for _ in range(2)]
    scales = [torch.full((1, 2, 1), math.nan, device=DEV) for _ in range(2)]
    for i in range(16):
        lens = torch.tensor([i], dtype=torch.int32, device=DEV)
        row = k[:, :, i:i + 1].to(DEV)
        co_alibi_cache_append_8bit(row, -row, *caches, *scales, lens)
        got = oracle.values(caches[0].cpu(), scales[0].cpu())[:, :, :i + 1]
        step = scales[0].cpu().double()[..., None]
        exact = k[:, :, :i + 1].double()
        bound = step if fmt == INT8 else torch.maximum(exact.abs() * 2.0 ** -4, step * 2.0 ** -9)
        assert ((got - exact).abs() <= bound).all()
        assert torch.equal(got, -oracle.values(caches[1].cpu(), scales[1].cpu())[:, :, :i + 1])


@FORMATS
def test_values_that_no_code_holds(fmt):
    """An infinity, a NaN, a scale past the last: the block's scale is NaN, the other blocks' and heads' are not, and stays so
    until the block is begun again."""
    k, v, caches, scales, table = make(2, 2, 40, 64, F32, fmt, 16, 64, seed=5)
    k[0, 0, 3, 5], v[1, 1, 20, 0], k[1, 0, 39, 63] = math.inf, math.nan, 1e30
    lens = torch.tensor([0, 7], dtype=torch.int32)
    c, s = run_and_check(k, v, caches, scales, table, lens)
    assert torch.isnan(s[0]).sum() == 2 and torch.isnan(s[1]).sum() == 1
    c, s = [t.cpu() for t in c], [t.cpu() for t in s]
    more = torch.randn(2, 2, 4, 64, generator=torch.Generator().manual_seed(6))
    # Sequence 0's block goes on; of sequence 1, rows 30 to 33 go on in the block of v's NaN and begin the one of k's at 32.
    c2, s2 = run_and_check(more, more, c, s, table, torch.tensor([9, 30], dtype=torch.int32))
    assert torch.isnan(s2[0]).sum() == 1 and torch.isnan(s2[1]).sum() == 1
    c2, s2 = run_and_check(more, more, c, s, table, torch.tensor([0, 16], dtype=torch.int32))
    assert torch.isnan(s2[0]).sum() == 1 and torch.isnan(s2[1]).sum() == 0


@FORMATS
def test_scales_from_elsewhere(fmt):
    """Scales that are no powers of two are doubled, too; ones that no block may have stay NaN."""
    k, v, caches, scales, table = make(3, 2, 5, 64, F32, fmt, 16, 64, seed=7)
    gen = torch.Generator().manual_seed(8)
    scales = [s * (1 + torch.rand(s.shape, generator=gen)) for s in scales]
    # (Quotients of fp32 values are rounded once before they are rounded to a code: keep them off the borders of codes.)
    want = oracle.append(k, v, caches, scales, torch.tensor([3, 16, 30]), table, None, None)
    c, s = [dev(t) for t in caches], [dev(t) for t in scales]
    co_alibi_cache_append_8bit(dev(k), dev(v), *c, *s, torch.tensor([3, 16, 30], device=DEV, dtype=torch.int32), block_table=dev(table))
    for got, exp in zip(s, want[1]):
        assert torch.allclose(got.cpu(), exp, rtol=2.0 ** -23, atol=0)
    for got, exp in zip(c, want[0]):
        assert same(got, exp)
    for bad in (0.0, -1.0, math.inf, math.nan, 2.0 ** -41, 2.0 ** 41):
        scales = [torch.full_like(x, bad) for x in scales]
        run_and_check(k, v, caches, scales, table, torch.tensor([3, 16, 30], dtype=torch.int32))


@FORMATS
def test_layouts(fmt):
    """Transposed and packed sources, an unaligned one, caches of one layer of several, int64 indices."""
    B, Hkv, T, D, page = 2, 3, 9, 64, 16
    k, v, caches, scales, table = make(B, Hkv, T, D, F16, fmt, page, 60, seed=2)
    lens = torch.tensor([3, 40], dtype=torch.int32)
    want, want_scales = oracle.append(k, v, caches, scales, lens, table, None, None)
    packed = torch.stack([k.transpose(1, 2), v.transpose(1, 2)], 2).to(DEV)
    odd = torch.empty(k.numel() + 1, dtype=F16, device=DEV)[1:].view(k.shape).copy_(k)
    layered = lambda t: torch.stack([t, t, t], 1)[:, 1]  # noqa: E731  (pages of other layers between)
    heads = lambda t: torch.cat([t, t], 1)[:, :t.shape[1]]  # noqa: E731
    for label, nk, nv, wrap in [("packed", packed[:, :, 0].transpose(1, 2), packed[:, :, 1].transpose(1, 2), lambda t: t),
                                ("unaligned", odd, v.to(DEV), lambda t: t), ("layers", k.to(DEV), v.to(DEV), layered),
                                ("heads", k.to(DEV), v.to(DEV), heads)]:
        c, s = [wrap(t.to(DEV).view(torch.uint8)).view(fmt) for t in caches], [wrap(t.to(DEV)) for t in scales]
        before = s[0]._version
        co_alibi_cache_append_8bit(nk, nv, *c, *s, lens.to(DEV).long(), block_table=table.to(DEV).long())
        for got, exp in zip((*c, *s), (*want, *want_scales)):
            assert torch.equal(got.contiguous().cpu().view(torch.uint8), exp.view(torch.uint8)), label
        assert s[0]._version > before
        assert all(same(a, b) for a, b in zip(
            co_alibi_cache_read_8bit(*c, *s, lens.to(DEV), 12, dtype=F32, block_table=table.to(DEV)),
            [x.float() for x in oracle.read(want, want_scales, lens, table, None, 12)])), label


@FORMATS
@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
@pytest.mark.parametrize("case", [
    # B, Hkv, D, page, capacity, rows
    (1, 1, 16, 0, 5, 5), (3, 2, 64, 16, 100, 37), (2, 3, 128, 0, 41, 41), (2, 2, 256, 64, 200, 1), (4, 1, 32, 256, 300, 300),
], ids=str)
def test_read_matches_oracle(case, dtype, fmt):
    B, Hkv, D, page, cap, rows = case
    _, _, caches, scales, table = make(B, Hkv, 1, D, dtype, fmt, page, cap, seed=D)
    gen = torch.Generator().manual_seed(rows)
    for first in (None, torch.randint(-3, cap, (B,), generator=gen, dtype=torch.int32)):
        lens = torch.randint(0, cap + 1, (B,), generator=gen, dtype=torch.int32)
        lens[0] = (cap, 1 << 30)[first is not None]
        want = oracle.read(caches, scales, lens, table, first, rows)
        got = co_alibi_cache_read_8bit(*map(dev, caches), *map(dev, scales), dev(lens), rows, dtype=dtype, block_table=dev(table),
                                       first=dev(first))
        for x, y in zip(got, want):
            assert x.dtype == dtype and x.is_contiguous() and torch.equal(x.cpu(), y.float().to(dtype))


def test_read_of_bad_pages_and_scales_is_nan():
    _, _, caches, scales, table = make(2, 2, 1, 64, F32, E4M3, 16, 48, seed=3)
    table[1, 1] = 1 << 30
    scales[0][int(table[0, 2]), 1, 0] = 0.0
    scales[1][int(table[0, 0]), 0, 0] = math.inf
    lens = torch.tensor([48, 40], dtype=torch.int32)
    got = co_alibi_cache_read_8bit(*map(dev, caches), *map(dev, scales), dev(lens), 48, dtype=F32, block_table=dev(table))
    for x, y in zip(got, oracle.read(caches, scales, lens, table, None, 48)):
        assert torch.equal(torch.isnan(x.cpu()), torch.isnan(y)) and torch.isnan(x).any()
        assert torch.equal(torch.nan_to_num(x.cpu()), torch.nan_to_num(y).float())


def test_rows_past_32_bits():
    """A pool of more than 2^32 bytes: its last pages are written and read like the first."""
    Hkv, D, page = 8, 128, 64
    pages = (1 << 32) // (Hkv * D * page) + 5
    caches = [torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.empty(pages, Hkv, page // 16, device=DEV) for _ in range(2)]
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, Hkv, 150, D, generator=gen).to(BF16) for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    co_alibi_cache_append_8bit(k.to(DEV), v.to(DEV), *caches, *scales, zero, block_table=table)
    got = co_alibi_cache_read_8bit(*caches, *scales, zero + 150, 150, dtype=F32, block_table=table)
    small = [torch.zeros(3, Hkv, page, D, dtype=torch.int8) for _ in range(2)]
    want = oracle.append(k, v, small, [torch.zeros(3, Hkv, 4) for _ in range(2)], [0], torch.tensor([[0, 1, 2]]), None, None)
    for x, y in zip(got, oracle.read(*want, [150], torch.tensor([[0, 1, 2]]), None, 150)):
        assert torch.equal(x.cpu(), y.float())


def test_empty_calls():
    k, v, caches, scales, table = make(2, 2, 3, 64, F16, INT8, 16, 32)
    k, v, table = k.to(DEV), v.to(DEV), table.to(DEV)
    c, s = [t.to(DEV) for t in caches], [t.to(DEV) for t in scales]
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    co_alibi_cache_append_8bit(k[:, :, :0], v[:, :, :0], *c, *s, lens, block_table=table)
    co_alibi_cache_append_8bit(k, v, *c, *s, lens, block_table=table, rows=torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    co_alibi_cache_append_8bit(k, v, *c, *s, lens, block_table=table[:, :0])
    assert all(same(a, b) for a, b in zip((*c, *s), (*caches, *scales)))
    out = co_alibi_cache_read_8bit(*c, *s, lens, 0, block_table=table)
    assert out[0].shape == (2, 2, 0, 64)
    out = co_alibi_cache_read_8bit(*c, *s, lens + 5, 3, block_table=table[:, :0])
    assert out[1].shape == (2, 2, 3, 64) and not out[1].any()


def test_captured_appends_and_reads():
    """A captured step that grows a cache, replayed with eager work between; the lengths move on the device."""
    gen = torch.Generator().manual_seed(1)
    k = torch.randn(2, 2, 40, 64, generator=gen).to(BF16)
    caches = [torch.zeros(2, 2, 64, 64, dtype=E4M3, device=DEV) for _ in range(2)]
    scales = [torch.zeros(2, 2, 4, device=DEV) for _ in range(2)]
    row, lens = torch.zeros(2, 2, 1, 64, dtype=BF16, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)

    def step():
        co_alibi_cache_append_8bit(row, row, *caches, *scales, lens)
        lens.add_(1)
        return co_alibi_cache_read_8bit(*caches, *scales, lens, 64, dtype=F32)

    step()
    lens.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lens.zero_()
    ref_c, ref_s = [torch.zeros(2, 2, 64, 64).to(E4M3) for _ in range(2)], [torch.zeros(2, 2, 4) for _ in range(2)]
    for i in range(40):
        row.copy_(k[:, :, i:i + 1])
        graph.replay()
        (torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)).sum()
        torch.cuda.synchronize()
        ref_c, ref_s = oracle.append(k[:, :, i:i + 1], k[:, :, i:i + 1], ref_c, ref_s, [i, i], None, None, None)
        want = oracle.read(ref_c, ref_s, [i + 1, i + 1], None, None, 64)
        assert torch.equal(out[0].cpu(), want[0].float()) and torch.equal(out[1].cpu(), want[1].float())


def test_another_stream():
    k, v, caches, scales, table = make(2, 2, 33, 128, BF16, INT8, 16, 90, seed=4)
    want, want_scales = oracle.append(k, v, caches, scales, [5, 20], table, None, None)
    c, s = [t.to(DEV) for t in caches], [t.to(DEV) for t in scales]
    lens = torch.tensor([5, 20], dtype=torch.int32, device=DEV)
    args = k.to(DEV), v.to(DEV), *c, *s, lens, table.to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        co_alibi_cache_append_8bit(*args)
        got = co_alibi_cache_read_8bit(*c, *s, lens + 33, 60, dtype=F32, block_table=table.to(DEV))
    side.synchronize()
    assert all(same(a, b) for a, b in zip(c, want)) and all(same_scales(a, b) for a, b in zip(s, want_scales))
    assert torch.equal(got[0].cpu(), oracle.read(want, want_scales, [38, 53], table, None, 60)[0].float())
