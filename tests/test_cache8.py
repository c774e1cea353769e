"""The 8-bit cache's and beam search's operators without a GPU: schemas, shape functions, argument checks of the Python functions
and of the C entry points, and the float64 oracle's own properties."""
import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import co_alibi_attn as co
from co_alibi_attn import _native
from oracle import serving as plain
from oracle import serving8 as oracle

P = 4096  # an aligned address that no accepted call may reach
E4M3 = torch.float8_e4m3fn


def test_operators_are_registered_with_their_schemas():
    ops = torch.ops.co_alibi
    assert str(ops.decode_tree_8bit.default._schema) == (
        "co_alibi::decode_tree_8bit(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor k_scale, "
        "Tensor v_scale, Tensor slopes, Tensor? seq_lens, Tensor? parents, Tensor? block_table, SymInt max_seq_len, "
        "float sm_scale, bool with_lse) -> (Tensor, Tensor)")
    assert str(ops.cache_append_8bit.default._schema) == (
        "co_alibi::cache_append_8bit(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor seq_lens, Tensor? counts, Tensor? rows, Tensor? block_table) -> ()")
    assert str(ops.cache_read_8bit.default._schema) == (
        "co_alibi::cache_read_8bit(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor seq_lens, "
        "Tensor? first, Tensor? block_table, SymInt rows, ScalarType dtype) -> (Tensor, Tensor)")
    assert str(ops.beam_select.default._schema) == (
        "co_alibi::beam_select(Tensor logits, Tensor scores, Tensor? finished, SymInt num_beams, SymInt end_token) -> "
        "(Tensor, Tensor, Tensor)")
    assert str(ops.cache_reorder.default._schema) == (
        "co_alibi::cache_reorder(Tensor(a!)[] caches, Tensor block_table, Tensor pages, Tensor seq_lens, Tensor parents, "
        "SymInt page_size) -> (Tensor, Tensor)")


def test_shapes_under_fake_tensors():
    with FakeTensorMode():
        cuda = dict(device="cuda")
        q = torch.empty(2, 8, 5, 64, dtype=torch.bfloat16, **cuda)
        k = torch.empty(2, 5, 2, 64, dtype=torch.bfloat16, **cuda).transpose(1, 2)
        pool = torch.empty(12, 2, 32, 64, dtype=E4M3, **cuda)
        scale = torch.empty(12, 2, 2, **cuda)
        table = torch.empty(2, 6, dtype=torch.int32, **cuda)
        lens = torch.empty(2, dtype=torch.int32, **cuda)
        o, lse = co.co_alibi_decode_tree_8bit(q, k, k, pool, pool, scale, scale, seq_len=lens, block_table=table, return_lse=True)
        assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (2, 8, 5) and lse.dtype == torch.float32
        assert co.co_alibi_cache_append_8bit(k, k, pool, pool.clone(), scale, scale.clone(), lens, block_table=table) is None
        x, y = co.co_alibi_cache_read_8bit(pool, pool, scale, scale, lens, 77, dtype=torch.float16, block_table=table)
        assert x.shape == y.shape == (2, 2, 77, 64) and x.dtype == torch.float16
        s, p, t = co.co_alibi_beam_select(torch.empty(3, 4, 100, **cuda), torch.empty(3, 4, **cuda), num_beams=6)
        assert s.shape == p.shape == t.shape == (3, 6)
        assert (s.dtype, p.dtype, t.dtype) == (torch.float32, torch.int32, torch.int64)
        new, n = co.co_alibi_cache_reorder([pool, scale], lens.long(), torch.empty(1, 2, dtype=torch.int64, **cuda), table, table)
        assert new.shape == table.shape and n.shape == (2,) and new.dtype == n.dtype == torch.int32


# ------------------------------------------------------------------ the C entry points


def _call(fn, defaults, over):
    unknown = set(over) - set(defaults)
    assert not unknown, unknown
    return getattr(_native.lib(), fn)(*{**defaults, **over}.values())


TREE = dict(dtype=1, fmt=0, q=P, k=P, v=P, kc=P, vc=P, ks=P, vs=P, strides=None, scale_strides=None, slopes=P, lens=None,
            parents=None, per_seq=0, table=None, blocks=0, pages=0, page=512, o=P, lse=None, ws=P, ws_bytes=1 << 50, B=2, Hq=8,
            Hkv=2, T=5, L=300, D=128, scale=0.125, stream=None)
APPEND = dict(dtype=1, fmt=0, k=P, v=P, kc=P, vc=P, ks=P, vs=P, strides=None, scale_strides=None, lens=P, counts=None, rows=None,
              n=5, table=None, blocks=0, pages=0, page=512, B=2, Hkv=2, T=5, D=128, stream=None)
READ = dict(dtype=1, fmt=0, kc=P, vc=P, ks=P, vs=P, strides=None, scale_strides=None, lens=P, first=None, rows=9, table=None,
            blocks=0, pages=0, page=512, k=P, v=P, B=2, Hkv=2, D=128, stream=None)
SELECT = dict(dtype=1, logits=P, strides=None, scores=P, finished=None, end=0, out=P, parents=P, tokens=P, ws=P,
              ws_bytes=1 << 50, B=2, W=4, N=4, V=1000, stream=None)


def longs(*x):
    return (ctypes.c_longlong * len(x))(*x)


def _strides(n, row=128):
    return longs(*([1 << 20, 1 << 15, row] * n))


@pytest.mark.parametrize("over,code,msg", [
    (dict(fmt=2), 2, "format must be 0 (e4m3) or 1 (int8)"),
    (dict(fmt=-1), 2, "format must be"),
    (dict(q=None), 1, "q is NULL"),
    (dict(k=8), 1, "k is not 16-byte aligned"),
    (dict(vc=None), 1, "v_cache is NULL"),
    (dict(ks=None), 1, "k_scale is NULL"),
    (dict(vs=2), 1, "v_scale is not 4-byte aligned"),
    (dict(scale_strides=longs(4, 1, -4, 1)), 1, "the strides of the scales must be >= 0"),
    (dict(strides=longs(*[1 << 20, 1 << 15, 128] * 3, 1 << 20, 1 << 15, 256, 1 << 20, 1 << 15, 256)), 1, "rows of an 8-bit cache must be dense"),
    (dict(strides=longs(*[1 << 20, 1 << 15, 128] * 3, 8, 1 << 15, 128, 8, 1 << 15, 128)), 1, "the strides of k_cache must be >= 0 and whole 16-byte"),
    (dict(L=513), 1, "seq_kv must be in [0, 512]"),
    (dict(table=P, blocks=4, pages=4, page=48), 1, "power of two >= 16, got 48"),
    (dict(T=65), 2, "at most 64 new tokens"),
    (dict(D=80), 2, "head_dim must be 16, 32, 64, 128 or 256"),
    (dict(D=256, dtype=0), 2, "head_dim 256 needs fp16 or bf16"),
    (dict(dtype=3), 2, "dtype must be"),
    (dict(scale=float("nan")), 1, "sm_scale must be finite"),
    (dict(L=900, page=1024, T=3, lens=P, ws_bytes=0), 1, "workspace of 0 bytes, need"),
    (dict(L=900, page=1024, T=3, lens=P, ws=None), 1, "workspace is NULL"),
    (dict(B=1 << 20, Hq=1 << 10, T=64), 1, "problem too large"),
])
def test_decode_tree_argument_errors(over, code, msg):
    assert _call("co_alibi_decode_tree_8bit", TREE, over) == code
    assert msg in _native.lib().co_alibi_last_error().decode()


@pytest.mark.parametrize("over,code,msg", [
    (dict(fmt=5), 2, "format must be"),
    (dict(n=0), 1, "new_rows must be >= 1"),
    (dict(n=6), 1, "new_rows is above tokens"),
    (dict(v=None), 1, "v is NULL"),
    (dict(lens=None), 1, "seq_lens is NULL"),
    (dict(vs=None), 1, "v_scale is NULL"),
    (dict(strides=longs(*[1 << 20, 1 << 18, 256] * 4)), 1, "must be dense"),
    (dict(strides=longs(1 << 20, 1 << 15, 128, 1 << 20, 1 << 15, 128, 0, 1 << 16, 128, 1 << 20, 1 << 16, 128)), 1, "the rows of k_cache overlap"),
    (dict(scale_strides=longs(64, 32, 16, 32)), 1, "the rows of v_scale overlap"),
    (dict(B=0), 1, ">= 1"),
    (dict(D=8), 2, "head_dim must be"),
    (dict(n=1 << 30, T=1 << 30), 1, "too large"),
])
def test_append_argument_errors(over, code, msg):
    assert _call("co_alibi_cache_append_8bit", APPEND, over) == code
    assert msg in _native.lib().co_alibi_last_error().decode()


@pytest.mark.parametrize("over,code,msg", [
    (dict(fmt=3), 2, "format must be"),
    (dict(dtype=7), 2, "dtype must be"),
    (dict(rows=0), 1, ">= 1"),
    (dict(k=8), 1, "k is not 16-byte aligned"),
    (dict(kc=None), 1, "k_cache is NULL"),
    (dict(first=1), 1, "first is not 4-byte aligned"),
    (dict(ks=None), 1, "k_scale is NULL"),
    (dict(strides=_strides(2, 512)), 1, "must be dense"),
    (dict(table=6, blocks=4, pages=4, page=64), 1, "block_table is not 4-byte aligned"),
    (dict(rows=1 << 30), 1, "too large"),
])
def test_read_argument_errors(over, code, msg):
    assert _call("co_alibi_cache_read_8bit", READ, over) == code
    assert msg in _native.lib().co_alibi_last_error().decode()


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=3), 2, "dtype must be"),
    (dict(B=0), 1, "batch must be >= 1"),
    (dict(W=65), 1, "beams and num_beams must be in [1, 64]"),
    (dict(N=0), 1, "beams and num_beams must be in [1, 64]"),
    (dict(V=(1 << 20) + 1), 1, "vocab must be in [1, 1048576]"),
    (dict(strides=longs(-1, 5)), 1, "the strides of logits must be >= 0"),
    (dict(finished=P, end=1000), 1, "end_token must be in [0, vocab)"),
    (dict(logits=1), 1, "logits is not 2-byte aligned"),
    (dict(scores=None), 1, "scores is NULL"),
    (dict(tokens=4), 1, "tokens is not 8-byte aligned"),
    (dict(ws_bytes=100), 1, "workspace of 100 bytes, need"),
    (dict(ws=P + 8), 1, "workspace is not 256-byte aligned"),
    (dict(B=1 << 30), 1, "too large"),
])
def test_select_argument_errors(over, code, msg):
    assert _call("co_alibi_beam_select", SELECT, over) == code
    assert msg in _native.lib().co_alibi_last_error().decode()


def test_select_workspace():
    size = _native.lib().co_alibi_beam_select_workspace_bytes
    assert size(1, 0, 1, 1, 9) == size(1, 1, 65, 1, 9) == size(1, 1, 1, 65, 9) == size(1, 1, 1, 1, 0) == 0
    for dtype, B, W, N, V in ((0, 1, 1, 1, 1), (0, 1, 4, 4, 50304), (2, 16, 8, 8, 131071)):
        assert 3 * 256 <= size(dtype, B, W, N, V) <= B * W * (-(-V // 1024) * (12 + 8 * N)) + 3 * 256


def _reorder(**over):
    a = dict(pools=[P], shape=[4096, 1024, 4, 64, 16], table=P, pages=P, lens=P, parents=P, out=P, out_lens=P, B=2, W=4, J=8,
             units=64, page=64)
    a.update(over)
    pools = (ctypes.c_void_p * len(a["pools"]))(*a["pools"]) if a["pools"] is not None else None
    shapes = longs(*a["shape"]) if a["shape"] is not None else None
    return _native.lib().co_alibi_cache_reorder(pools, shapes, 1, a["table"], a["pages"], a["lens"], a["parents"], a["out"],
                                                a["out_lens"], a["B"], a["W"], a["J"], a["units"], a["page"], None)


@pytest.mark.parametrize("over,msg", [
    (dict(B=0), ">= 1"),
    (dict(J=0), ">= 1"),
    (dict(W=65), "beams must be in [1, 64]"),
    (dict(page=24), "power of two >= 16, got 24"),
    (dict(B=1 << 20, J=1 << 12), "too large"),
    (dict(J=1 << 25), "too large"),
    (dict(pools=None), "pools or shapes is NULL"),
    (dict(shape=None), "pools or shapes is NULL"),
    (dict(pools=[2]), "pool 0 is not 4-byte aligned"),
    (dict(table=None), "block_table is NULL"),
    (dict(parents=1), "parents is not 4-byte aligned"),
    (dict(shape=[4096, 1024, 4, 48, 16]), "entries that divide a page's rows"),
    (dict(shape=[4096, 1024, 4, 128, 8]), "entries that divide a page's rows"),
    (dict(shape=[4096, 1024, 4, 64, 6]), "entries of whole 4 bytes"),
    (dict(shape=[4096, 1000, 4, 64, 16]), "do not overlap"),
    (dict(shape=[4000, 1024, 4, 64, 16]), "do not overlap"),
    (dict(shape=[4098, 1024, 4, 64, 16]), "whole 4 bytes apart"),
    (dict(shape=[1 << 40, 1 << 30, 1 << 10, 64, 1 << 20]), "too large"),
])
def test_reorder_argument_errors(over, msg):
    assert _reorder(**over) == 1
    assert msg in _native.lib().co_alibi_last_error().decode()


# ------------------------------------------------------------------ the Python functions


def test_python_refusals():
    """CPU tensors are refused where they have to be, and everything that the types and shapes can tell before a launch."""
    with FakeTensorMode():
        cuda = dict(device="cuda")
        q = torch.empty(2, 4, 3, 64, dtype=torch.bfloat16, **cuda)
        k = torch.empty(2, 2, 3, 64, dtype=torch.bfloat16, **cuda)
        c, s = torch.empty(2, 2, 40, 64, dtype=torch.int8, **cuda), torch.empty(2, 2, 3, **cuda)
        lens = torch.empty(2, dtype=torch.int32, **cuda)
        tree = lambda *a, **kw: co.co_alibi_decode_tree_8bit(*a, **kw)  # noqa: E731
        for bad, error in (((q, k, k, c.float(), c.float(), s, s), TypeError), ((q, k, k, c, c.view(E4M3), s, s), TypeError),
                           ((q, k, k, c, c, s.half(), s), TypeError), ((q, k, k, c, c, s[:, :, :2], s), ValueError),
                           ((q, k, k, c, c[:, :, :30], s, s), ValueError), ((q, k, k.half(), c, c, s, s), TypeError),
                           ((q[:, :3], k, k, c, c, s, s), AssertionError), ((q, k, k, c, c, s.cpu(), s), AssertionError),
                           ((q[..., :40], k[..., :40], k[..., :40], c, c, s, s), ValueError)):
            with pytest.raises(error):
                tree(*bad)
        for kw in (dict(seq_len=41), dict(seq_len=-1), dict(seq_len=lens, max_seq_len=41), dict(seq_len=lens[:1]),
                   dict(block_table=torch.empty(3, 2, dtype=torch.int32, **cuda))):
            with pytest.raises(ValueError):
                tree(q, k, k, c, c, s, s, **kw)
        append = lambda *a, **kw: co.co_alibi_cache_append_8bit(*a, **kw)  # noqa: E731
        with pytest.raises(TypeError):
            append(k, k, c.half(), c.half(), s, s, lens)
        with pytest.raises(ValueError):
            append(k[0], k[0], c, c, s, s, lens)
        with pytest.raises(ValueError):
            append(k, k, c, c, s.clone().requires_grad_(), s, lens)
        read = lambda *a, **kw: co.co_alibi_cache_read_8bit(*a, **kw)  # noqa: E731
        with pytest.raises(TypeError):
            read(c, c, s, s, lens, 4, dtype=torch.int8)
        for bad in (-1, 2.5):
            with pytest.raises(ValueError):
                read(c, c, s, s, lens, bad)
        x, y = torch.empty(2, 4, 100, **cuda), torch.empty(2, 4, **cuda)
        select = lambda *a, **kw: co.co_alibi_beam_select(*a, **kw)  # noqa: E731
        for bad, error in (((x[0], y), ValueError), ((x, y[:, :3]), ValueError), ((x.double(), y), TypeError),
                           ((x, y.half()), TypeError), ((x.cpu(), y), AssertionError)):
            with pytest.raises(error):
                select(*bad)
        for kw, error in ((dict(num_beams=0), ValueError), (dict(num_beams=65), ValueError),
                          (dict(finished=y), TypeError), (dict(finished=y[:, :2] > 0), ValueError),
                          (dict(finished=y > 0, end_token=100), ValueError), (dict(finished=y > 0, end_token=-1), ValueError)):
            with pytest.raises(error):
                select(x, y, **kw)
        table, par = torch.empty(4, 3, dtype=torch.int32, **cuda), torch.empty(2, 2, dtype=torch.int32, **cuda)
        four, pool = torch.empty(4, dtype=torch.int32, **cuda), torch.empty(9, 2, 16, 64, **cuda)
        for bad, error in ((([], four, par, table, table), ValueError), (([pool[0, 0]], four, par, table, table), ValueError),
                           (([pool], four, par[0], table, table), ValueError), (([pool.cpu()], four, par, table, table), AssertionError),
                           (([pool.clone().requires_grad_()], four, par, table, table), ValueError)):
            with pytest.raises(error):
                co.co_alibi_cache_reorder(*bad)


# ------------------------------------------------------------------ the oracle


@pytest.mark.parametrize("fmt", (E4M3, torch.int8), ids=("e4m3", "int8"))
def test_oracle_codes(fmt):
    """torch's own conversions, and the scales' definition."""
    most = oracle.LARGEST[fmt]
    x = torch.cat([torch.linspace(-most, most, 4001).double(), torch.arange(-20, 20) / 1024.0, torch.tensor([2.0 ** -10, 3 * 2.0 ** -10])])
    want = x.float().to(E4M3).double() if fmt == E4M3 else torch.round(x)
    assert torch.equal(oracle.code(x, fmt), want)
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, 2, 20, 32, generator=gen, dtype=torch.float64).float() for _ in range(2))
    caches, scales = oracle.append(k, v, [torch.zeros(1, 2, 32, 32).to(fmt)] * 2, [torch.zeros(1, 2, 2)] * 2, [0], None, None, None)
    for x, c, s in zip((k, v), caches, scales):
        for h in range(2):
            for i in range(2):
                top = float(x[0, h, 16 * i:16 * i + 16].abs().max())
                assert math.log2(float(s[0, h, i])).is_integer() and top <= most * float(s[0, h, i]) < 2 * top
        err = (oracle.values(c, s)[:, :, :20] - x.double()).abs()
        step = s.double().repeat_interleave(16, 2)[:, :, :20, None]
        assert (err <= (step / 2 if fmt == torch.int8 else torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10))).all()


def test_oracle_decode_is_the_plain_one_over_the_values():
    gen = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(1, 4, 3, 32, generator=gen), torch.randn(1, 2, 3, 32, generator=gen), torch.randn(1, 2, 3, 32, generator=gen)
    caches = [torch.randint(-127, 128, (1, 2, 40, 32), generator=gen, dtype=torch.int8) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-8, -5, (1, 2, 3), generator=gen).float()) for _ in range(2)]
    lam = torch.tensor([1.0, 0.5, 0.25, 0.1])
    got = oracle.decode_tree(q, k, v, caches, scales, [37], None, None, lam, 0.2)
    kc, vc = (oracle.values(c, s) for c, s in zip(caches, scales))
    want = plain.decode_tree(q, k, v, kc, vc, [37], None, None, lam, 0.2)
    assert torch.allclose(got[0], want[0], rtol=1e-12) and torch.allclose(got[1], want[1], rtol=1e-12)


def test_oracle_select_is_a_sort():
    gen = torch.Generator().manual_seed(2)
    x, s = torch.randn(2, 3, 50, generator=gen), torch.randn(2, 3, generator=gen)
    got = oracle.beam_select(x, s, 7)
    best, at = (torch.log_softmax(x.double(), 2) + s.double()[..., None]).view(2, -1).sort(1, descending=True)
    assert torch.allclose(torch.tensor(got[0], dtype=torch.float64), best[:, :7], rtol=1e-12)
    assert got[1] == (at[:, :7] // 50).tolist() and got[2] == (at[:, :7] % 50).tolist()
