"""co_alibi_sample against the float64 oracle: tokens are equal.  Needs an MI355X.

Both sides add up float64 weights, the kernel as integers of 2^-46 of the largest at 50304 tokens, so a
uniform number would have to lie within about 1e-9 of a border between two tokens for them to differ.
"""
import math

import pytest
import torch

from co_alibi_attn import co_alibi_sample
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = (F32, BF16, F16)


def logits_of(B, V, dtype, seed, scale=2.5, masked=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=gen) * scale
    if masked:
        x.masked_fill_(torch.rand(B, V, generator=gen) < masked, -math.inf)
    return x.to(dtype), torch.rand(B, generator=gen)


def run(x, u, t=1.0, k=0, p=1.0, m=0.0):
    got = co_alibi_sample(x.to(DEV), u.to(DEV), temperature=t, top_k=k, top_p=p, min_p=m)
    assert got.dtype == torch.int64 and got.shape == x.shape[:1]
    return got.tolist()


def check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    B = x.shape[0]
    assert run(x, u, t, k, p, m) == oracle.sample(x, u, [t] * B, [k] * B, [p] * B, [m] * B)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", (1, 2, 63, 64, 65, 1000, 1023, 5000, 50304))
def test_settings(V, dtype):
    x, u = logits_of(16, V, dtype, seed=V)
    for kw in (dict(), dict(t=0.7), dict(t=3.0), dict(k=1), dict(k=5), dict(k=40), dict(k=V), dict(k=V + 7), dict(p=0.9),
               dict(p=0.3), dict(p=1e-9), dict(m=0.05), dict(m=1.0), dict(t=0.0), dict(t=0.8, k=50, p=0.95, m=0.02),
               dict(t=1.5, k=max(1, V // 2), p=0.8), dict(t=1e-3), dict(t=1e30), dict(p=0.0)):
        print(V, dtype, kw, flush=True)
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ties_go_to_the_lowest_index(dtype):
    gen = torch.Generator().manual_seed(3)
    x = torch.randint(-3, 4, (12, 3000), generator=gen).to(dtype)  # a few hundred tokens of every value
    u = torch.rand(12, generator=gen)
    for kw in (dict(), dict(t=0.0), dict(k=7), dict(k=900), dict(p=0.5), dict(k=1500, p=0.77), dict(m=0.3)):
        check(x, u, **kw)
    flat = torch.zeros(4, 50304, dtype=dtype)  # all equal: the u * V-th token
    u = torch.tensor([0.0, 0.25, 0.5, 0.999])
    assert run(flat, u) == [math.floor(float(v) * 50304) for v in u]
    assert run(flat, u, k=10) == [math.floor(float(v) * 10) for v in u]
    assert run(flat, u, p=0.5) == [math.floor(float(v) * 25152) for v in u]
    zeros = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], dtype=dtype)  # signed zeros are equal
    assert [run(zeros, torch.tensor([v]))[0] for v in (0.0, 0.3, 0.6, 0.9)] == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_special_rows(dtype):
    inf, nan = math.inf, math.nan
    low = torch.finfo(dtype).min
    rows = torch.tensor([[0, 1, 2, 3], [nan, 1, 2, 3], [0, 1, 2, nan], [-inf] * 4, [inf, 1, inf, 2], [-inf, -inf, 5, -inf],
                         [low, low, low, low], [low, 0, -inf, low], [inf, -inf, nan, 0], [-inf, inf, -inf, -inf],
                         [3, 3, -inf, -inf]], dtype=dtype)
    for u in (0.0, 0.3, 0.6, 0.999):
        for kw in (dict(), dict(t=0.0), dict(k=2), dict(k=3), dict(p=0.6), dict(m=0.5), dict(t=2.0)):
            check(rows, torch.full((11,), u), **kw)


@pytest.mark.parametrize("dtype", (F32, BF16), ids=str)
def test_cuts_of_many_tokens_and_cuts_together(dtype):
    x, u = logits_of(6, 50304, dtype, seed=21)
    for kw in (dict(k=700), dict(k=800), dict(k=801), dict(k=2047), dict(k=2049, p=0.9), dict(k=50303), dict(p=0.999999),
               dict(p=0.9, m=1e-4), dict(p=0.2, m=1e-4), dict(p=0.999, m=0.3), dict(m=1e-6), dict(m=1e-300), dict(k=30, m=0.2),
               dict(k=5000, m=1e-3, p=0.7), dict(t=20.0, m=0.5), dict(t=20.0, p=0.5), dict(t=0.05), dict(t=0.02, p=0.5)):
        print(dtype, kw, flush=True)
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_tokens_close_together(dtype):
    """Rows whose tokens crowd into few distances, alone, with masked ones and with one far below."""
    x, u = logits_of(6, 60000, dtype, seed=23, scale=0.05)
    masked = x.masked_fill(torch.rand(x.shape, generator=torch.Generator().manual_seed(24)) < 0.3, -math.inf)
    outlier = x.clone()
    outlier[:, 777] = -30000.0
    for rows in (x, masked, outlier, x.abs().clamp(max=0.02)):
        for kw in (dict(), dict(k=20000, p=0.9), dict(p=0.5, t=1.3), dict(t=0.01), dict(k=59999)):
            print(dtype, kw, flush=True)
            check(rows, u, **kw)


def test_temperatures_and_logits_of_any_size():
    x, u = logits_of(6, 5000, F32, seed=22)
    wide = x * 1e37  # up to about 1e38
    tiny = x * 1e-42  # subnormal
    for rows in (x, wide, tiny):
        for t in (1e-300, 1e-40, 1e-6, 1e6, 1e40, 1e300, math.inf):
            for kw in (dict(), dict(k=20), dict(p=0.5), dict(m=0.5), dict(m=1.0)):
                print(t, kw, flush=True)
                check(rows, u, t=t, **kw)


def test_masked_vocabulary():
    for dtype in DTYPES:
        x, u = logits_of(8, 20011, dtype, seed=5, masked=0.9)
        for kw in (dict(), dict(k=100), dict(k=10000), dict(p=0.9), dict(m=0.01)):
            check(x, u, **kw)
            picked = run(x, u, **kw)
            assert torch.isfinite(x[torch.arange(8), picked]).all()


def test_uniforms():
    x, _ = logits_of(1, 777, F32, seed=6)
    x = x.expand(9, 777)
    u = torch.tensor([0.0, 1e-30, 0.25, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, math.nan, math.inf])
    check(x, u, p=0.9)
    u64 = torch.linspace(0, 1, 9, dtype=torch.float64)
    check(x, u64, k=300)
    assert run(x[:1], torch.tensor([1.0 - 2.0 ** -53], dtype=torch.float64)) == run(x[:1], torch.tensor([1.0]))


def test_settings_per_row():
    B = 32
    x, u = logits_of(B, 3001, BF16, seed=8)
    gen = torch.Generator().manual_seed(9)
    t = torch.rand(B, generator=gen) * 2
    t[::7] = 0.0
    t[3] = math.nan
    t[4] = -1.0
    t[5] = math.inf
    k = torch.randint(-1, 100, (B,), generator=gen, dtype=torch.int32)
    p = torch.rand(B, generator=gen) * 1.2
    p[6], p[8] = -1.0, math.nan
    m = torch.rand(B, generator=gen) * 0.3 - 0.1
    m[10], m[11] = 1.5, math.nan
    want = oracle.sample(x, u, t.tolist(), k.tolist(), p.tolist(), m.tolist())
    assert run(x, u, t.to(DEV), k.to(DEV), p.to(DEV), m.to(DEV)) == want
    assert run(x, u, t.to(DEV), k.long().to(DEV), p.to(DEV), m.to(DEV)) == want
    assert run(x, u, t.double().to(DEV), k.to(DEV), p.to(DEV), 0.0) == oracle.sample(x, u, t.tolist(), k.tolist(), p.tolist(),
                                                                                   [0.0] * B)


@pytest.mark.parametrize("seed", range(10))
def test_random(seed):
    gen = torch.Generator().manual_seed(seed)
    B, V = int(torch.randint(1, 33, (1,), generator=gen)), int(torch.randint(1, 9000, (1,), generator=gen))
    dtype = DTYPES[seed % 3]
    x, u = logits_of(B, V, dtype, seed=seed, scale=(0.01, 1.0, 4.0, 20.0)[seed % 4], masked=0.3 * (seed % 2))
    t = torch.rand(B, generator=gen) * 1.5
    k = torch.randint(0, V + 1, (B,), generator=gen, dtype=torch.int32)
    p, m = torch.rand(B, generator=gen), torch.rand(B, generator=gen) * 0.1
    want = oracle.sample(x, u, t.tolist(), k.tolist(), p.tolist(), m.tolist())
    assert run(x, u, t.to(DEV), k.to(DEV), p.to(DEV), m.to(DEV)) == want


def test_layouts_and_large_vocabularies():
    x, u = logits_of(5, 4001, F16, seed=11)
    want = run(x, u, p=0.9)
    wide = torch.full((5, 5000), 99.0, dtype=F16)
    wide[:, 3:4004] = x
    got = co_alibi_sample(wide.to(DEV)[:, 3:4004], u.to(DEV), top_p=0.9)  # rows apart, odd alignment
    assert got.tolist() == want
    assert co_alibi_sample(x.to(DEV).t().contiguous().t(), u.to(DEV), top_p=0.9).tolist() == want  # not dense rows
    assert co_alibi_sample(x.to(DEV)[:1].expand(5, 4001), u.to(DEV), top_p=0.9).tolist() == run(x[:1].expand(5, 4001), u, p=0.9)
    assert co_alibi_sample(x.to(DEV)[:0], u.to(DEV)[:0]).shape == (0,)
    big, u = logits_of(2, 1 << 20, F32, seed=12)
    check(big, u, p=0.95)
    check(big, u, k=70000)


def test_refusals_on_the_device():
    x, u = torch.randn(3, 9, device=DEV), torch.rand(3, device=DEV)
    with pytest.raises(ValueError, match="top_k must be one value"):
        co_alibi_sample(x, u, top_k=torch.ones(2, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError, match="int32 or int64"):
        co_alibi_sample(x, u, top_k=torch.ones(3, device=DEV))
    with pytest.raises(TypeError, match="uniforms must be float32 or float64"):
        co_alibi_sample(x, u.half())
    with pytest.raises(ValueError, match="logits must be"):
        co_alibi_sample(torch.empty(1, (1 << 20) + 1, device=DEV, dtype=F16), u[:1])


def test_capture_and_other_streams():
    x, u = logits_of(4, 50304, BF16, seed=13)
    x, u = x.to(DEV), u.to(DEV)
    want = co_alibi_sample(x, u, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = co_alibi_sample(x, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = co_alibi_sample(x, u, top_p=0.9)
    for i in range(4):
        x.neg_()
        u.mul_(0.8)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, co_alibi_sample(x, u, top_p=0.9)), i
