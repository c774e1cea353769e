"""co_alibi_beam_select and co_alibi_cache_reorder against the float64 oracle (oracle/serving8.py).  Needs an MI355X.

Parents and tokens have to be equal (random scores lie far further apart than the 2^-22 that fp32 exponentials leave).  Scores:
log S is off by the exponentials' 2^-22 of themselves at most, and the score is rounded to fp32 once.
"""
import math

import pytest
import torch

from co_alibi_attn import co_alibi_beam_select, co_alibi_cache_reorder
from oracle import serving8 as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def check(logits, scores, n, finished=None, end_token=0, got=None):
    want = oracle.beam_select(logits, scores, n, finished, end_token)
    if got is None:
        got = co_alibi_beam_select(logits.to(DEV), scores.to(DEV), num_beams=n, end_token=end_token,
                                   finished=None if finished is None else finished.to(DEV))
    s, p, t = (x.cpu() for x in got)
    assert s.dtype == F32 and p.dtype == torch.int32 and t.dtype == torch.int64
    assert p.tolist() == want[1] and t.tolist() == want[2]
    ws = torch.tensor(want[0], dtype=torch.float64)
    dead = ws == -math.inf
    assert torch.equal(s == -math.inf, dead)
    assert ((s.double() - ws).abs() <= 2.0 ** -22 + 2.0 ** -24 * ws.abs())[~dead].all()
    return s, p, t


def draw(B, W, V, dtype, seed=0, scale=2.5):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(B, W, V, generator=gen) * scale).to(dtype), -20 * torch.rand(B, W, generator=gen), gen


@pytest.mark.parametrize("dtype", (F32, BF16, F16), ids=str)
@pytest.mark.parametrize("case", [
    # B, W, N, V
    (1, 1, 1, 1), (1, 4, 4, 50304), (3, 1, 5, 50304), (2, 8, 8, 4097), (5, 3, 64, 100), (1, 64, 64, 300), (2, 2, 7, 131071),
    (40, 16, 4, 1000), (1, 2, 33, 1023), (2, 5, 5, 1024), (1, 1, 64, 63), (1, 1, 2, 1 << 20),
], ids=str)
def test_select_matches_oracle(case, dtype):
    B, W, N, V = case
    logits, scores, _ = draw(B, W, V, dtype, seed=V)
    check(logits, scores, N)


@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_ties(dtype):
    """Equal logits go by token, equal beams by beam: a constant row, few values, twins, more ties than a list holds."""
    logits, scores, gen = draw(2, 4, 20000, dtype, seed=1)
    logits[0, 0] = 0.5
    logits[0, 1] = torch.randint(0, 3, (20000,), generator=gen).to(dtype)
    logits[0, 3] = logits[0, 2]
    scores[0] = torch.tensor([-1.0, -1.0, -2.0, -2.0])
    logits[1] = -3.0
    scores[1] = -5.0
    for n in (1, 4, 50):
        check(logits, scores, n)
    flat = torch.zeros(1, 2, 9000, dtype=dtype)
    check(flat, torch.zeros(1, 2), 64)
    few = torch.full((1, 2, 9000), -math.inf, dtype=dtype)
    few[0, 0, [17, 8999]], few[0, 1, 4000] = 1.0, 2.0
    check(few, torch.zeros(1, 2), 5)


def test_logits_that_64_bits_cannot_tell_apart():
    """Far below the row's largest, different logits score the same: the larger one still comes first."""
    logits = torch.full((1, 1, 300), -math.inf)
    logits[0, 0, 0] = 1e4
    logits[0, 0, 1:] = torch.arange(299) * 1e-20
    s, p, t = (x.cpu() for x in co_alibi_beam_select(logits.to(DEV), torch.zeros(1, 1, device=DEV), num_beams=5))
    assert t.tolist() == [[0, 299, 298, 297, 296]]


def test_rows_without_candidates():
    """NaN, no logit above -inf, +inf, scores that are not finite: whole rows and whole sequences of them."""
    logits, scores, _ = draw(4, 4, 5000, F32, seed=2)
    logits[0, 1, 4999] = math.nan
    logits[0, 2] = -math.inf
    scores[0, 3] = -math.inf
    logits[1, 0, [3, 70, 4000]] = math.inf
    scores[1, 1:] = torch.tensor([math.nan, math.inf, -math.inf])
    logits[2] = math.nan
    logits[3, 2, 1:] = -math.inf
    for n in (1, 4, 9):
        s, p, t = check(logits, scores, n)
        assert (s[2] == -math.inf).all() and (p[2] == 0).all() and (t[2] == -1).all()
    logits, scores, _ = draw(1, 2, 3, F16, seed=3)  # fewer tokens than places
    s, p, t = check(logits, scores, 8)
    assert (t[0, 6:] == -1).all() and (t[0, :6] >= 0).all()


def test_finished_beams():
    logits, scores, gen = draw(3, 6, 2000, BF16, seed=4)
    finished = torch.rand(3, 6, generator=gen) < 0.5
    finished[1] = True
    logits[finished] = math.nan  # not read
    for end, n in ((0, 6), (1999, 3), (7, 12)):
        check(logits, scores, n, finished, end)
    scores[1, 2] = -math.inf
    check(logits, scores, 6, finished, 5)


def test_layouts_and_streams():
    logits, scores, _ = draw(2, 4, 5001, F32, seed=5)
    wide = torch.zeros(2, 4, 3, 5010, device=DEV)
    wide[:, :, 1, 3:5004] = logits.to(DEV)
    check(logits, scores, 4, got=co_alibi_beam_select(wide[:, :, 1, 3:5004], scores.to(DEV)))
    swapped = logits.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    check(logits, scores, 4, got=co_alibi_beam_select(swapped, scores.to(DEV)))
    strange = logits.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    on = scores.to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = co_alibi_beam_select(strange, on)
    side.synchronize()
    check(logits, scores, 4, got=got)
    assert [x.shape for x in co_alibi_beam_select(wide[:0, :, 0], on[:0], num_beams=3)] == [(0, 3)] * 3


def test_select_is_the_same_every_time_and_under_capture():
    logits, scores, _ = draw(3, 4, 50304, BF16, seed=6)
    x, s = logits.to(DEV), scores.to(DEV)
    first = co_alibi_beam_select(x, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = co_alibi_beam_select(x, s)
    for i in range(5):
        x.copy_(logits.roll(i, 2))
        graph.replay()
        eager = co_alibi_beam_select(x, s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(out, first))


# ------------------------------------------------------------------ reordering


def pools_of(num_pages, H, page, D, dtype, gen, layers=2):
    out = []
    for _ in range(2 * layers):
        x = torch.randint(0, 256, (num_pages, H, page, D * torch.empty(0, dtype=dtype).element_size()), generator=gen, dtype=torch.uint8)
        out.append(x if dtype == torch.uint8 else x.view(dtype))
    out += [torch.randn(num_pages, H, page // 16, generator=gen) for _ in range(2 * layers)]
    return out


def raw(t):
    return t.cpu().contiguous().view(torch.uint8)


@pytest.mark.parametrize("case", [
    # B, W, J, H, page, D, dtype
    (1, 1, 2, 1, 16, 16, torch.uint8), (1, 4, 3, 12, 64, 64, BF16), (3, 5, 4, 2, 16, 32, torch.uint8), (2, 64, 2, 1, 16, 16, F32),
    (4, 8, 5, 3, 32, 128, torch.int8), (2, 3, 1, 2, 256, 16, F16),
], ids=str)
def test_reorder_matches_oracle(case):
    """Steps of a search: rows are appended (random bytes), beams reordered; tables, lengths and every byte are compared, and
    every sequence holds the rows of its ancestors."""
    B, W, J, H, page, D, dtype = case
    gen = torch.Generator().manual_seed(W)
    num_pages = B * W * J + 3
    caches = pools_of(num_pages, H, page, D, dtype, gen)
    pages = torch.randperm(num_pages, generator=gen)[:B * W * J].view(B * W, J).to(torch.int32)
    table = pages.clone()
    lens = torch.zeros(B * W, dtype=torch.int32)
    told = [[] for _ in range(B * W)]  # the first pool's rows as they were written
    dc = [t.to(DEV) for t in caches]
    for step in range(12):
        n = int(torch.randint(0, max(2, page * J // 8), (1,), generator=gen))
        for i in range(B * W):
            g = i // W
            for _ in range(n + (g % 2)):  # groups of different lengths
                r = int(lens[i])
                if r == page * J:
                    break
                u = int(table[i, r // page])
                for t in caches[:4]:
                    x = torch.randint(0, 256, t[u, :, r % page].view(torch.uint8).shape, generator=gen, dtype=torch.uint8)
                    t[u, :, r % page] = x.view(t.dtype)
                told[i].append(raw(caches[0][u, :, r % page]))
                lens[i] += 1
        parents = torch.randint(0, W, (B, W), generator=gen)
        if step % 3 == 0:
            parents = parents.sort(1).values
        if step == 5:
            parents[:, 0], parents[:, -1] = -4, W + 9  # clamped
        dc = [t.to(DEV) for t in caches]
        want = oracle.reorder(caches, table, pages, lens, parents, page)
        new_table, new_lens = co_alibi_cache_reorder(dc, lens.to(DEV), parents.to(DEV), table.to(DEV), pages.to(DEV))
        torch.cuda.synchronize()
        assert torch.equal(new_table.cpu(), want[1]) and torch.equal(new_lens.cpu(), want[2])
        for i, (a, b) in enumerate(zip(dc, want[0])):
            assert torch.equal(raw(a), raw(b)), (step, i)
        par = parents.clamp(0, W - 1)
        told = [list(told[g * W + int(par[g, i])]) for g in range(B) for i in range(W)]
        caches, table, lens = want
        for i in range(B * W):
            assert int(lens[i]) == len(told[i])
            for r in ({0, len(told[i]) // 2, len(told[i]) - 1} if told[i] else ()):
                assert torch.equal(raw(caches[0][int(table[i, r // page]), :, r % page]), told[i][r])
            # What is not full is nobody else's.
            g = i // W
            others = torch.cat([table[g * W:i], table[i + 1:g * W + W]])
            for j in range(int(lens[i]) // page, J):
                assert not (others[:, j] == table[i, j]).any()


def test_reorder_of_bad_tables_stays_inside_the_pool():
    """Entries outside the pool are moved as they are, and no copy is made from or to them; lengths past the capacity are full."""
    gen = torch.Generator().manual_seed(0)
    caches = pools_of(8, 2, 16, 16, torch.uint8, gen, layers=1)
    pages = torch.arange(8, dtype=torch.int32).view(4, 2)
    table = torch.tensor([[0, 1], [2, -1], [1 << 30, 5], [6, 7]], dtype=torch.int32)
    lens = torch.tensor([20, 20, 5, 1 << 29], dtype=torch.int32)
    parents = torch.tensor([[1, 1, 2, 2]])
    dc = [t.to(DEV) for t in caches]
    got = co_alibi_cache_reorder(dc, lens.to(DEV), parents.to(DEV), table.to(DEV), pages.to(DEV))
    want = oracle.reorder(caches, table, pages, lens, parents, 16)
    assert torch.equal(got[0].cpu(), want[1]) and torch.equal(got[1].cpu(), want[2])
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(dc, want[0]))
    got = co_alibi_cache_reorder(dc, lens.to(DEV), torch.full((1, 4), 3, device=DEV), table.to(DEV), pages.to(DEV))
    assert got[0].cpu().tolist() == [[6, 7]] * 4 and got[1].cpu().tolist() == [1 << 29] * 4
    got = co_alibi_cache_reorder(dc, -lens.to(DEV), parents.to(DEV), table.to(DEV), pages.to(DEV))
    assert got[0].cpu().tolist() == pages.tolist()  # nothing is filled: everyone gets pages of their own


def test_many_pools_and_strided_ones():
    """More pools than one launch takes, layers of one buffer, pools of 4-byte rows, unaligned ones."""
    gen = torch.Generator().manual_seed(1)
    B, W, J, H, page = 2, 3, 2, 2, 16
    n = B * W * J
    pages = torch.randperm(n, generator=gen).view(B * W, J).to(torch.int32)
    lens = torch.full((B * W,), 21, dtype=torch.int32)
    parents = torch.tensor([[2, 2, 2], [0, 2, 0]])
    layers = torch.randint(0, 256, (n, 70, H, page, 16), generator=gen, dtype=torch.uint8)
    odd = torch.randint(0, 256, (n * H * page * 4 + 4,), generator=gen, dtype=torch.uint8)
    host = [layers[:, i] for i in range(70)] + [odd[4:].view(n, H, page, 4)]
    want = oracle.reorder(host, pages, pages, lens, parents, page)
    on, on_odd = layers.to(DEV), odd.to(DEV)
    pools = [on[:, i] for i in range(70)] + [on_odd[4:].view(n, H, page, 4)]
    before = pools[0]._version
    got = co_alibi_cache_reorder(pools, lens.to(DEV).long(), parents.to(DEV), pages.to(DEV).long(), pages.to(DEV))
    assert torch.equal(got[0].cpu(), want[1]) and torch.equal(got[1].cpu(), want[2]) and pools[0]._version > before
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(pools, want[0]))
    assert on_odd[:4].cpu().tolist() == odd[:4].tolist()


def test_reorder_captured():
    gen = torch.Generator().manual_seed(2)
    B, W, J, page = 2, 4, 3, 16
    caches = pools_of(B * W * J, 2, page, 16, BF16, gen)
    dc = [t.to(DEV) for t in caches]
    pages = torch.arange(B * W * J, dtype=torch.int32).view(B * W, J)
    table, lens = pages.to(DEV), torch.zeros(B * W, dtype=torch.int32, device=DEV)
    home, parents = table.clone(), torch.zeros(B, W, dtype=torch.int32, device=DEV)

    def step():
        t, n = co_alibi_cache_reorder(dc, lens, parents, table, home)
        table.copy_(t)
        lens.copy_(n)
        lens.add_(5)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    ht, hl = pages.clone(), torch.full((B * W,), 5, dtype=torch.int32)
    caches = [t.cpu() for t in dc]
    for i in range(7):
        par = torch.randint(0, W, (B, W), generator=gen)
        parents.copy_(par)
        graph.replay()
        torch.cuda.synchronize()
        caches, ht, hl = oracle.reorder(caches, ht, pages, hl, par, page)
        hl += 5
        assert torch.equal(table.cpu(), ht) and torch.equal(lens.cpu(), hl)
        assert all(torch.equal(raw(a), raw(b)) for a, b in zip(dc, caches))


def test_every_pool_is_looked_at():
    pool, par = torch.zeros(4, 2, 16, 64, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    table, lens = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2), torch.tensor([5, 0], dtype=torch.int32, device=DEV)
    for bad in (pool.clone().requires_grad_(), pool.cpu(), pool[:3], pool.transpose(2, 3)):
        with pytest.raises(ValueError):
            co_alibi_cache_reorder([pool, bad], lens, par, table, table)


def test_pools_and_logits_past_32_bits():
    page, H, D = 64, 8, 128
    pages = (1 << 32) // (page * H * D) + 8
    pool = torch.zeros(pages, H, page, D, dtype=torch.int8, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(7)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device=DEV).view(2, 2)
    tail = torch.randint(-127, 128, (4, H, page, D), generator=gen, device=DEV, dtype=torch.int8)
    pool[-4:] = tail
    lens = torch.tensor([70, 3], dtype=torch.int32, device=DEV)
    new, n = co_alibi_cache_reorder([pool], lens, torch.zeros(1, 2, dtype=torch.int32, device=DEV), table, table)
    assert n.tolist() == [70, 70] and new.tolist() == [[pages - 4, pages - 3], [pages - 4, pages - 1]]
    assert torch.equal(pool[-1, :, :6], tail[1, :, :6]) and torch.equal(pool[-1, :, 6:], tail[3, :, 6:])
    assert torch.equal(pool[-4:-1], tail[:3]) and not pool[:4].any() and not pool[-8:-4].any()
    del pool
    W, V = 64, 1 << 20
    logits = torch.zeros(35, W, V, dtype=BF16, device=DEV)
    logits[-1] = torch.randn(W, V, generator=gen, device=DEV).to(BF16)
    scores = torch.randn(35, W, generator=gen, device=DEV)
    got = co_alibi_beam_select(logits, scores, 5)
    want = co_alibi_beam_select(logits[-1:].clone(), scores[-1:].clone(), 5)
    for x, y in zip(got, want):
        assert torch.equal(x[-1:], y)
    assert got[2][0].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("B,W,N,V,dtype", [(2, 16, 32, 50304, BF16), (1, 16, 31, 9000, F32), (3, 5, 17, 20000, F16), (1, 3, 64, 1000, F32),
                                           (1, 64, 40, 262144, BF16)])
def test_many_of_many(B, W, N, V, dtype):
    """Rounds of the ranking, and the end of them; the last one has more lists than a round."""
    logits, scores, _ = draw(B, W, V, dtype, seed=9)
    check(logits, scores * 0.05, N)


@pytest.mark.parametrize("N", (9, 32, 64))
def test_ties_among_many(N):
    """A few different logits, and beams of equal scores: every order but the scores' counts."""
    logits = torch.randint(0, 3, (2, 8, 20000), generator=torch.Generator().manual_seed(N)).float()
    logits[:, 1::2] = logits[:, ::2]
    check(logits, torch.zeros(2, 8), N)
    check(logits.flip(2).to(BF16), torch.zeros(2, 8), N)
