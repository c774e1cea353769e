"""The serving step's operators without a GPU: schemas, shape functions, argument checks of the Python
functions and of the C entry points, and the float64 oracle's own properties."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import co_alibi_attn as co
from co_alibi_attn import _native
from co_alibi_attn.gpt import GPT, GPTConfig, PagedCache
from oracle import co_alibi_ref as ref
from oracle import serving as oracle

P = 4096  # an aligned address that no accepted call may reach


def test_operators_are_registered_with_their_schemas():
    tree = str(torch.ops.co_alibi.decode_tree.default._schema)
    append = str(torch.ops.co_alibi.cache_append.default._schema)
    sample = str(torch.ops.co_alibi.sample.default._schema)
    assert tree == ("co_alibi::decode_tree(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor slopes, "
                    "Tensor? seq_lens, Tensor? parents, Tensor? block_table, SymInt max_seq_len, float sm_scale, "
                    "bool with_lse) -> (Tensor, Tensor)")
    assert append == ("co_alibi::cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, "
                      "Tensor seq_lens, Tensor? counts, Tensor? rows, Tensor? block_table) -> ()")
    assert sample == ("co_alibi::sample(Tensor logits, Tensor uniforms, Tensor? temperature, Tensor? top_k, "
                      "Tensor? top_p, Tensor? min_p, float temperature_all, SymInt top_k_all, float top_p_all, "
                      "float min_p_all) -> Tensor")


def test_shapes_under_fake_tensors():
    with FakeTensorMode():
        q = torch.empty(2, 8, 5, 64, device="cuda", dtype=torch.bfloat16)
        k = torch.empty(2, 5, 2, 64, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
        pool = torch.empty(12, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
        table = torch.empty(2, 6, device="cuda", dtype=torch.int32)
        lens = torch.empty(2, device="cuda", dtype=torch.int32)
        o, lse = co.co_alibi_decode_tree(q, k, k, pool, pool, seq_len=lens, block_table=table, return_lse=True)
        assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous()
        assert lse.shape == (2, 8, 5) and lse.dtype == torch.float32
        assert co.co_alibi_cache_append(k, k, pool, pool.clone(), lens, block_table=table) is None
        tokens = co.co_alibi_sample(torch.empty(3, 100, device="cuda"), torch.empty(3, device="cuda"))
        assert tokens.shape == (3,) and tokens.dtype == torch.int64


def _tree(lib, **over):
    a = dict(dtype=1, q=P, k=P, v=P, kc=P, vc=P, strides=None, slopes=P, lens=None, parents=None, per_seq=0, table=None,
             blocks=0, pages=0, page=512, o=P, lse=None, ws=P, ws_bytes=1 << 50, B=2, Hq=8, Hkv=2, T=5, L=300, D=128,
             scale=0.125)
    a.update(over)
    return lib.co_alibi_decode_tree(a["dtype"], a["q"], a["k"], a["v"], a["kc"], a["vc"], a["strides"], a["slopes"],
                                    a["lens"], a["parents"], a["per_seq"], a["table"], a["blocks"], a["pages"], a["page"],
                                    a["o"], a["lse"], a["ws"], a["ws_bytes"], a["B"], a["Hq"], a["Hkv"], a["T"], a["L"],
                                    a["D"], a["scale"], None)


def _strides(n, row=128):
    return (ctypes.c_longlong * (3 * n))(*([1 << 20, 1 << 15, row] * n))


@pytest.mark.parametrize("over,code,msg", [
    (dict(q=None), 1, "q is NULL"),
    (dict(k=8), 1, "k is not 16-byte aligned"),
    (dict(vc=None), 1, "v_cache is NULL"),
    (dict(slopes=None), 1, "slopes is NULL"),
    (dict(parents=2), 1, "parents is not 4-byte aligned"),
    (dict(lens=2), 1, "seq_lens is not 4-byte aligned"),
    (dict(table=6, blocks=4, pages=4, page=64), 1, "block_table is not 4-byte aligned"),
    (dict(table=P, blocks=40, pages=4, page=8), 1, "power of two >= 16, got 8"),
    (dict(table=P, blocks=40, pages=4, page=48), 1, "power of two >= 16, got 48"),
    (dict(table=P, blocks=0, pages=4, page=64), 1, "blocks_per_seq and num_pages must be >= 1"),
    (dict(table=P, blocks=4, pages=4, page=64), 1, "seq_kv must be in [0, 256]"),
    (dict(L=513), 1, "seq_kv must be in [0, 512]"),
    (dict(L=-1), 1, "seq_kv must be in [0, 512]"),
    (dict(page=0), 1, "page_size must be >= 1"),
    (dict(T=65), 2, "at most 64 new tokens"),
    (dict(T=0), 1, ">= 1"),
    (dict(Hq=6, Hkv=4), 1, "multiple of heads_kv"),
    (dict(D=80), 2, "head_dim must be 16, 32, 64, 128 or 256"),
    (dict(D=256, dtype=0), 2, "head_dim 256 needs fp16 or bf16"),
    (dict(dtype=3), 2, "dtype must be"),
    (dict(scale=float("nan")), 1, "sm_scale must be finite"),
    (dict(strides=_strides(5, 100)), 1, "the strides of q must be >= 0 and whole 16-byte units"),
    (dict(strides=_strides(5, 64)), 1, "the row stride of q must be in"),
    (dict(strides=_strides(5, 1 << 21)), 1, "the row stride of q must be in"),
])
def test_decode_tree_argument_errors(over, code, msg):
    lib = _native.lib()
    assert _tree(lib, **over) == code
    assert msg in lib.co_alibi_last_error().decode()


def test_decode_tree_workspace():
    """Per sequence and kv head one int, then per (sequence, query head, token, split) three floats and D more, each
    array rounded up to 256 bytes; nothing with one split."""
    lib = _native.lib()
    size = lambda *a: lib.co_alibi_decode_tree_workspace_bytes(*a)  # noqa: E731
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    for dtype, B, Hq, Hkv, T, L, D in ((1, 1, 4, 4, 1, 900, 64), (2, 2, 8, 2, 16, 5000, 128), (0, 1, 6, 2, 3, 9000, 32)):
        n = size(dtype, B, Hq, Hkv, T, L, D)
        rows = B * Hq * T
        for splits in range(2, 513):
            if n == up(4 * B * Hkv) + 3 * up(4 * rows * splits) + 4 * rows * splits * D:
                break
        else:
            raise AssertionError((n, rows))
        assert splits <= -(-L // 64) + 1
    assert size(1, 1, 4, 4, 1, 0, 64) == 0 and size(1, 1, 4, 4, 1, 300, 64) == 0  # few chunks: one split
    for bad in ((1, 0, 4, 4, 1, 9, 64), (1, 1, 2, 4, 1, 9, 64), (1, 1, 4, 4, 0, 9, 64), (1, 1, 4, 4, 1, -1, 64)):
        assert size(*bad) == 0
    need = size(2, 2, 8, 2, 3, 500, 128)
    assert need > 0
    for over, msg in ((dict(ws=None, ws_bytes=need), "workspace is NULL"), (dict(ws=P + 16, ws_bytes=need), "workspace is not 256"),
                      (dict(lens=P, ws_bytes=need - 1), f"workspace of {need - 1} bytes, need {need}")):
        args = dict(dtype=2, B=2, Hq=8, Hkv=2, T=3, L=500, D=128)
        assert _tree(lib, **args, **over) == 1
        assert msg in lib.co_alibi_last_error().decode()


def test_cache_of_the_gpt_without_a_device():
    cfg = GPTConfig(n_layer=2, n_head=2, d_model=64, vocab=11)
    cache = PagedCache(cfg, 3, 70, torch.float32, "cpu", page_size=32)
    assert cache.capacity == 96 and cache.block_table.tolist() == [[0, 1, 2], [3, 4, 5], [6, 7, 8]]
    assert len(cache.layers) == 2 and cache.layers[0][0].shape == (9, 2, 32, 32)
    with pytest.raises(ValueError, match="no new keys"):
        cache.accept()
    cache.seq_lens += torch.tensor([5, 60, 0])
    cache.bound = 96
    cache.room_for(36)
    assert cache.bound == 60
    with pytest.raises(ValueError, match="37 more rows behind 60 do not fit a cache of 96"):
        cache.room_for(37)
    with pytest.raises(ValueError, match="empty cache"):
        GPT(cfg).prefill(torch.zeros(3, 4, dtype=torch.long), cache)


def _append(lib, **over):
    a = dict(dtype=2, k=P, v=P, kc=P, vc=P, strides=None, lens=P, counts=None, rows=None, n=5, table=None, blocks=0, pages=0,
             page=512, B=2, H=2, T=5, D=64)
    a.update(over)
    return lib.co_alibi_cache_append(a["dtype"], a["k"], a["v"], a["kc"], a["vc"], a["strides"], a["lens"], a["counts"],
                                     a["rows"], a["n"], a["table"], a["blocks"], a["pages"], a["page"], a["B"], a["H"],
                                     a["T"], a["D"], None)


@pytest.mark.parametrize("over,code,msg", [
    (dict(k=None), 1, "k is NULL"),
    (dict(kc=8), 1, "k_cache is not 16-byte aligned"),
    (dict(lens=None), 1, "seq_lens is NULL"),
    (dict(rows=2), 1, "rows is not 4-byte aligned"),
    (dict(n=6), 1, "new_rows is above tokens"),
    (dict(n=0), 1, "new_rows must be >= 1"),
    (dict(T=0), 1, ">= 1"),
    (dict(table=P, blocks=4, pages=4, page=24), 1, "power of two >= 16, got 24"),
    (dict(table=P, blocks=1 << 20, pages=4, page=2048), 1, "problem too large"),
    (dict(D=48), 2, "head_dim must be"),
    (dict(dtype=5), 2, "dtype must be"),
    (dict(strides=(ctypes.c_longlong * 12)(*[640, 320, 64] * 2, *[0, 32768, 64] * 2)), 1, "the rows of k_cache overlap"),
])
def test_cache_append_argument_errors(over, code, msg):
    lib = _native.lib()
    assert _append(lib, **over) == code
    assert msg in lib.co_alibi_last_error().decode()


def _sample(lib, **over):
    a = dict(dtype=0, logits=P, stride=100, uni=P, f64=0, t=None, k=None, p=None, m=None, out=P, B=2, V=100)
    a.update(over)
    return lib.co_alibi_sample(a["dtype"], a["logits"], a["stride"], a["uni"], a["f64"], a["t"], a["k"], a["p"], a["m"], 1.0, 0,
                               1.0, 0.0, a["out"], a["B"], a["V"], None)


@pytest.mark.parametrize("over,code,msg", [
    (dict(logits=None), 1, "logits is NULL"),
    (dict(logits=2), 1, "logits is not 4-byte aligned"),
    (dict(uni=4, f64=1), 1, "uniforms is not 8-byte aligned"),
    (dict(out=4), 1, "tokens is not 8-byte aligned"),
    (dict(t=2), 1, "temperature is not 4-byte aligned"),
    (dict(B=0), 1, "batch must be >= 1"),
    (dict(V=0), 1, "vocab must be in [1, 1048576]"),
    (dict(V=(1 << 20) + 1), 1, "vocab must be in [1, 1048576]"),
    (dict(stride=-1), 1, "row_stride must be >= 0"),
    (dict(dtype=9), 2, "dtype must be"),
])
def test_sample_argument_errors(over, code, msg):
    lib = _native.lib()
    assert _sample(lib, **over) == code
    assert msg in lib.co_alibi_last_error().decode()


def test_python_checks():
    q, k = torch.randn(1, 4, 2, 64), torch.randn(1, 2, 2, 64)
    kc = torch.randn(1, 2, 16, 64)
    with pytest.raises(ValueError, match=r"\(B, Hq, T, D\)"):
        co.co_alibi_decode_tree(q[0], k, k, kc, kc)
    with pytest.raises(AssertionError):
        co.co_alibi_decode_tree(q, k, k[:, :, :1], kc, kc)
    with pytest.raises(AssertionError, match="CUDA"):
        co.co_alibi_decode_tree(q, k, k, kc, kc)
    with pytest.raises(ValueError, match="at most 64 new tokens"):
        co.co_alibi_decode_tree(q[:, :, :1].expand(1, 4, 65, 64), *[k[:, :, :1].expand(1, 2, 65, 64)] * 2, kc, kc)
    with pytest.raises(ValueError, match=r"\(B, Hkv, T, D\)"):
        co.co_alibi_cache_append(k[0], k[0], kc, kc, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(AssertionError, match="CUDA"):
        co.co_alibi_cache_append(k, k, kc, kc, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="logits must be"):
        co.co_alibi_sample(torch.randn(5), torch.rand(5))
    with pytest.raises(ValueError, match=r"uniforms must be \(2,\)"):
        co.co_alibi_sample(torch.randn(2, 5), torch.rand(3))
    with pytest.raises(AssertionError, match="CUDA"):
        co.co_alibi_sample(torch.randn(2, 5), torch.rand(2))


def test_python_checks_of_values():
    with FakeTensorMode():
        def dev(*shape, dtype=torch.float16):
            return torch.empty(*shape, device="cuda", dtype=dtype)

        q, k, kc = dev(2, 4, 3, 64), dev(2, 2, 3, 64), dev(2, 2, 32, 64)
        lens = dev(2, dtype=torch.int32)
        for kw, msg in [(dict(seq_len=33), r"seq_len must be in \[0, 32\]"), (dict(seq_len=-1), "seq_len must be in"),
                        (dict(seq_len=lens, max_seq_len=33), r"max_seq_len must be in \[0, 32\]"),
                        (dict(seq_len=dev(3, dtype=torch.int32)), "per-sequence lengths"),
                        (dict(seq_len=dev(2)), "per-sequence lengths"),
                        (dict(block_table=dev(3, 4, dtype=torch.int32)), r"block_table must be \(2, blocks\)")]:
            with pytest.raises(ValueError, match=msg):
                co.co_alibi_decode_tree(q, k, k, kc, kc, **kw)
        with pytest.raises(TypeError, match="share one dtype"):
            co.co_alibi_decode_tree(q, k, k, kc.float(), kc)
        with pytest.raises(ValueError, match="head_dim must be one of"):
            co.co_alibi_decode_tree(dev(1, 1, 1, 48), *[dev(1, 1, 1, 48)] * 2, *[dev(1, 1, 9, 48)] * 2)
        with pytest.raises(ValueError, match="needs float16 or bfloat16"):
            f = torch.float32
            co.co_alibi_decode_tree(dev(1, 1, 1, 256, dtype=f), *[dev(1, 1, 1, 256, dtype=f)] * 2,
                                    *[dev(1, 1, 9, 256, dtype=f)] * 2)
        with pytest.raises(ValueError, match="cannot require gradients"):
            co.co_alibi_cache_append(k, k, kc.requires_grad_(), kc, lens)
        x, u = dev(2, 9), dev(2, dtype=torch.float32)
        for kw, msg in [(dict(temperature=-1.0), "temperature must be in"), (dict(temperature=float("nan")), "temperature"),
                        (dict(top_k=-1), "top_k must be in"), (dict(top_p=1.5), "top_p must be in"),
                        (dict(min_p=-0.1), "min_p must be in")]:
            with pytest.raises(ValueError, match=msg):
                co.co_alibi_sample(x, u, **kw)
        with pytest.raises(TypeError, match="logits must be float32"):
            co.co_alibi_sample(dev(2, 9, dtype=torch.float64), u)


# ------------------------------------------------------------------ the oracle's own properties


def test_oracle_tree_is_the_attention_oracle_on_each_chain():
    g = torch.Generator().manual_seed(0)
    B, Hq, Hkv, T, L, D, page = 2, 4, 2, 5, 21, 16, 16
    q = torch.randn(B, Hq, T, D, generator=g)
    k, v = torch.randn(B, Hkv, T, D, generator=g), torch.randn(B, Hkv, T, D, generator=g)
    kc, vc = torch.randn(B * 2, Hkv, page, D, generator=g), torch.randn(B * 2, Hkv, page, D, generator=g)
    table = torch.tensor([[3, 0], [1, 2]])
    parents = [[-1, 0, 0, 1, -1], [-1, -1, 5, 2, 1]]
    lens = [L, 9]
    lam = ref.slopes(Hq, 8.0).float()
    o, lse, _, _ = oracle.decode_tree(q, k, v, kc, vc, lens, parents, table, lam, 0.25)
    for b in range(B):
        for t in range(T):
            path = oracle.chain_of(parents[b], t)
            if path is None:
                assert (b, t) in ((1, 2), (1, 3)) and not o[b, :, t].any() and torch.isneginf(lse[b, :, t]).all()
                continue
            keys = torch.cat([oracle.gather_rows(kc, table, b, lens[b]), k[b][:, path]], 1)
            vals = torch.cat([oracle.gather_rows(vc, table, b, lens[b]), v[b][:, path]], 1)
            ro, rlse = ref.forward(q[b:b + 1, :, t:t + 1], keys[None], vals[None], lam, causal=False, scale=0.25)
            torch.testing.assert_close(o[b, :, t].float(), ro[0, :, 0], rtol=1e-5, atol=1e-5)
            torch.testing.assert_close(lse[b, :, t].float(), rlse[0, :, 0], rtol=1e-5, atol=1e-5)


def test_oracle_sample_known_draws():
    x = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]]))
    draw = lambda u, t=1.0, k=0, p=1.0, m=0.0: oracle.sample(x, [u], [t], [k], [p], [m])[0]  # noqa: E731
    assert [draw(u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91, 1.0)] == [1, 1, 3, 3, 2, 2, 0, 0]
    assert [draw(u, k=2) for u in (0.0, 0.56, 0.58, 0.999)] == [1, 1, 3, 3]  # 4/7 of the kept weight is token 1's
    assert [draw(u, p=0.5) for u in (0.0, 0.56, 0.58)] == [1, 1, 3]
    assert draw(0.999, p=0.39) == 1 and draw(0.999, m=0.74) == 3 and draw(0.999, m=0.76) == 1
    assert draw(0.9, t=0.0) == 1
    assert oracle.sample(torch.tensor([[1.0, 2.0, 2.0], [float("nan"), 0, 0], [-torch.inf] * 3]), [0.6] * 3, [0.0] * 3,
                         [0] * 3, [1.0] * 3, [0.0] * 3) == [1, -1, -1]
