"""What co_alibi_decode_tree may leave out of a sum: with the tail skip on cached keys below 2^-40 of it (fp32: 2^-64),
with the skip off nothing.  Needs an MI355X.

Tolerances: the oracle's first-order bound (oracle/serving.py) and half a step of the type.
"""
import math

import pytest
import torch

from co_alibi_attn import _native, co_alibi_decode_tree
from oracle import co_alibi_ref as ref
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
NAME = {torch.float16: "fp16", torch.bfloat16: "bf16", torch.float32: "fp32"}


def run(q, k, v, kc, vc, L, **kw):
    o = co_alibi_decode_tree(*(t.to(DEV) for t in (q, k, v, kc, vc)), seq_len=L, **kw)
    torch.cuda.synchronize()
    return o.cpu()


@pytest.mark.parametrize("dtype", NAME, ids=NAME.get)
@pytest.mark.parametrize("T", (1, 16, 40), ids=lambda t: f"rows{4 * t}")
@pytest.mark.parametrize("L", (120, 5000))
def test_without_the_tail_skip_every_value_is_read(L, T, dtype):
    """An infinity among the oldest values reaches every row, though its keys' weights are too small for fp32, from a
    split of its own as within one."""
    gen = torch.Generator().manual_seed(L + T)
    n = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k, v, kc, vc = n(1, 4, T, 64), n(1, 1, T, 64), n(1, 1, T, 64), n(1, 1, L, 64), n(1, 1, L, 64)
    lam = ref.slopes(4, 8.0, dtype=dtype).float()
    want, _, bound, _ = oracle.decode_tree(q, k, v, kc, vc, [L], None, None, lam, 0.125)
    vc[0, 0, 7, 5] = math.inf
    with _native.tail_skip(False):
        o = run(q, k, v, kc, vc, L)
    assert not torch.isfinite(o[..., 5]).any(), int(torch.isfinite(o[..., 5]).sum())
    rest = [d for d in range(64) if d != 5]
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * half if dtype == torch.float16 else 0.0
    over = (o.double() - want).abs() - (half * (want.abs() + bound) + bound + tiny)
    assert over[..., rest].max() <= 0


def test_a_key_heavier_than_its_splits_scale_counts():
    """A split's scale follows its maximum loosely: one key may weigh 2^11 times what the scale says.  Here the scale lies
    2^-64.5 below the row's and the key 2^-53.5, with a value of 2^55."""
    B, Hkv, L, D = 64, 2, 1024, 64
    low, heavy = -64.5 * math.log(2), -53.5 * math.log(2)
    gen = torch.Generator().manual_seed(1)
    q = torch.zeros(B, Hkv, 1, D)
    q[..., 0] = 8.0  # the score is the key's first element (scale 1/8)
    k, v = torch.zeros(B, Hkv, 1, D), torch.randn(B, Hkv, 1, D, generator=gen)
    kc, vc = torch.zeros(B, Hkv, L, D), torch.randn(B, Hkv, L, D, generator=gen)
    lam = ref.slopes(Hkv, 8.0).float()
    for row in (40, 200, 300, 450, 700):
        kc[..., 0] = low
        kc[:, :, row, 0] = heavy
        value = vc.clone()
        value[:, :, row, 9] = 2.0 ** 55
        want, _, bound, _ = oracle.decode_tree(q[:1], k[:1], v[:1], kc[:1], value[:1], [L], None, None, lam, 0.125)
        assert (want[..., 9] - v[:1, :, :, 9].double()).abs().min() > 1
        o = run(q, k, v, kc, value, L, sm_scale=0.125)
        over = (o[:1].double() - want).abs() - (2.0 ** -24 * (want.abs() + bound) + bound)
        assert over.max() <= 0, (row, over.max())


@pytest.mark.parametrize("dtype", NAME, ids=NAME.get)
@pytest.mark.parametrize("T", (1, 16, 40), ids=lambda t: f"rows{4 * t}")
def test_a_new_tokens_own_value_counts_however_light(T, dtype):
    """Only cached keys may be left out: a NaN among a token's own values shows, though its key's score is 100 below the
    cached ones'."""
    L = 5000
    gen = torch.Generator().manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k, v, kc, vc = n(1, 4, T, 64), n(1, 1, T, 64), n(1, 1, T, 64), n(1, 1, L, 64), n(1, 1, L, 64)
    q[..., 0], k[..., 0], kc[..., 0] = 1.0, -800.0, 0.0
    parents = torch.full((T,), -1, dtype=torch.int32)
    v[:, :, T // 2, 5] = math.nan
    o = run(q, k, v, kc, vc, L, parents=parents.to(DEV))
    assert o[:, :, T // 2, 5].isnan().all()
    o[:, :, T // 2, 5] = 0.0
    assert torch.isfinite(o).all()
