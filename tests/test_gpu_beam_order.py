"""co_alibi_beam_select: beams whose logits and scores are equal keep their order wherever their rows lie.  Needs an MI355X.

Rows of an odd vocabulary, and views, begin at different places within 16 bytes; equal rows have to get equal scores, bit for bit,
so that the lower beam comes first (and is the one that stays where only one of them can).
"""
import pytest
import torch

from co_alibi_attn import co_alibi_beam_select
from oracle import serving8 as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", (F32, BF16, F16), ids=str)


def row(V, dtype, seed):
    return (torch.randn(V, generator=torch.Generator().manual_seed(seed)) * 2.5).to(dtype)


def in_order(got, x, score, W, N):
    """W beams of the logits x: candidates by score, beam and token, and one score for all of a token's beams."""
    s, p, t = (y.cpu() for y in got)
    one = oracle.beam_select(x[None, None], torch.tensor([[score]]), min(N, x.numel()))
    want = sorted((-c, w, k) for c, k in zip(one[0][0], one[2][0]) for w in range(W))[:N]
    assert list(zip(p[0].tolist(), t[0].tolist())) == [f[1:] for f in want]
    for i in range(1, N):
        assert want[i][0] != want[i - 1][0] or s[0, i] == s[0, i - 1]


@DTYPES
@pytest.mark.parametrize("V", (131071, 50257, 100003, 4099, 1027, 517, 9, 5, 2))
def test_equal_beams_of_an_odd_vocabulary(V, dtype):
    for seed in range(3):
        x = row(V, dtype, seed)
        for W, N in ((8, 8), (8, 3), (5, min(20, 5 * V))):
            logits = x.expand(1, W, V).contiguous().to(DEV)
            in_order(co_alibi_beam_select(logits, torch.full((1, W), -3.7, device=DEV), N), x, -3.7, W, N)


@DTYPES
def test_equal_beams_in_rows_of_any_alignment(dtype):
    V, W = 20011, 8
    x = row(V, dtype, 7)
    for stride in (V, V + 1, V + 2, V + 3, V + 5, V + 8):
        for shift in (0, 1, 3):
            buffer = torch.zeros(1, W, stride + 16, dtype=dtype, device=DEV).view(-1)
            logits = buffer[shift:].as_strided((1, W, V), (W * stride, stride, 1))
            logits.copy_(x)
            in_order(co_alibi_beam_select(logits, torch.zeros(1, W, device=DEV), 12), x, 0.0, W, 12)


@DTYPES
def test_a_sequence_gives_the_same_wherever_it_lies(dtype):
    """The sequences of a batch, whose first rows lie differently: the same inputs give the same bits."""
    V, W, B = 5001, 3, 8
    gen = torch.Generator().manual_seed(1)
    x, scores = (torch.randn(1, W, V, generator=gen) * 2.5).to(dtype), -torch.rand(1, W, generator=gen)
    got = co_alibi_beam_select(x.expand(B, W, V).contiguous().to(DEV), scores.expand(B, W).contiguous().to(DEV), 9)
    for out in got:
        assert torch.equal(out, out[:1].expand_as(out))
