"""co_alibi_beam_select's sums where the exponentials' errors do not cancel: many equal logits far below the largest.  Needs an MI355X.

log S may be off by 2^-22: a weight's exponential by 2^-23 of itself (one step of its instruction), its reduced argument by three
roundings of 2^-25, in powers of two, which is 2^-24 of the weight; sums and powers of two are exact or fp64.  The score is rounded to fp32 once more:
2^-24 of itself.
"""
import math

import pytest
import torch

from co_alibi_attn import co_alibi_beam_select
from oracle import serving8 as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def check(logits, scores, n, ties=True):
    want = oracle.beam_select(logits, scores, n)
    s, p, t = (x.cpu() for x in co_alibi_beam_select(logits.to(DEV), scores.to(DEV), n))
    ws = torch.tensor(want[0], dtype=torch.float64)
    dead = ws == -math.inf
    assert torch.equal(s == -math.inf, dead)
    over = ((s.double() - ws).abs() - (2.0 ** -22 + 2.0 ** -24 * ws.abs()))[~dead]
    assert over.max() <= 0, f"scores off by {over.max():.2e} beyond their bound"
    if ties:
        assert p.tolist() == want[1] and t.tolist() == want[2]


@pytest.mark.parametrize("V,far", [(1 << 20, 12.05), (1 << 20, 13.5), (131072, 7.5), (131072, 11.0), (131071, 9.3), (50304, 10.7),
                                   (50257, 5.21), (20000, 3.3), (300, 5.6), (1 << 20, 17.0)], ids=str)
@pytest.mark.parametrize("dtype", (F32, BF16, F16), ids=str)
def test_one_peak_over_equal_logits(V, far, dtype):
    """One logit at 0, the others at -far; then all of it 3.7 and -61.3 further up (what a type can hold of it)."""
    for up in (0.0, 3.7, -61.3):
        logits = torch.full((1, 1, V), up - far).to(dtype)
        logits[0, 0, V // 3] = torch.tensor(up).to(dtype)
        check(logits, torch.zeros(1, 1), 1)


@pytest.mark.parametrize("shift", (1e3, -2.5e4, 6e4, -1e6, 1.5e6, 3e7, -1e9))
def test_rows_far_from_zero(shift):
    """Logits of large size, of which fp32 holds whole numbers or less: on both sides of 2^20, where the reference changes."""
    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(1, 3, 30011, generator=gen) * 3 + shift
    logits[0, 2] = shift + 2.0
    logits[0, 2, 1:] = shift - 6.0
    check(logits, -torch.rand(1, 3, generator=gen), 7)


def test_maxima_on_both_sides_of_the_reference():
    """A row whose parts' maxima lie below and above 2^20 in size, close to one another; huge spreads; the lowest number as a mask."""
    top = 2.0 ** 20
    logits = torch.full((1, 5, 40000), -3e38)
    logits[0, 0, ::2] = top - 1
    logits[0, 0, 20000:] = top + 0.5
    logits[0, 1] = -top - 0.25
    logits[0, 1, 30000:] = -top + 0.5
    logits[0, 2, 5], logits[0, 2, 39999] = 3e38, 2.9e38
    logits[0, 3] = torch.finfo(F32).min
    logits[0, 3, ::3] = 1.25
    logits[0, 4] = -math.inf
    logits[0, 4, 1000:3000] = -80.0
    check(logits, torch.zeros(1, 5), 1)
    for w in range(5):
        check(logits[:, w:w + 1], torch.zeros(1, 1), 2)


def test_wide_spreads():
    """Logits over tens of units with several scales of weight, in every type."""
    gen = torch.Generator().manual_seed(5)
    for dtype in (F32, BF16, F16):
        for scale in (0.3, 8.0, 30.0):
            check((torch.randn(2, 3, 50257, generator=gen) * scale).to(dtype), -3 * torch.rand(2, 3, generator=gen), 6)


def test_infinite_and_missing_numbers():
    """+inf counts, NaN and -inf in far places, in the segments of a long row."""
    logits = torch.full((1, 6, 100003), -4.0)
    logits[0, 0, [5, 70000, 100002]] = math.inf
    logits[0, 1, 99999] = math.nan
    logits[0, 2] = -math.inf
    logits[0, 3, 50000:] = -math.inf
    logits[0, 4, :99000] = -math.inf
    logits[0, 5, ::2] = torch.finfo(F32).min
    check(logits, torch.zeros(1, 6), 20)


@pytest.mark.parametrize("dtype", (F32, BF16, F16), ids=str)
def test_a_sole_candidate_scores_what_its_beam_does(dtype):
    """One token, or one that a mask leaves: log_softmax is 0 exactly, whatever the logit is, and beams of one score go in order; so do
    those with the same number of equal logits."""
    gen = torch.Generator().manual_seed(11)
    for V in (1, 2, 9, 1000, 50257):
        logits = torch.full((2, 16, V), -math.inf)
        where = torch.randint(0, V, (2, 16, 1), generator=gen)
        logits.scatter_(2, where, torch.randn(2, 16, 1, generator=gen) * torch.tensor([1.0, 300.0]).view(2, 1, 1))
        scores = -torch.randint(0, 3, (2, 16), generator=gen).float() * 0.7
        s, p, t = (x.cpu() for x in co_alibi_beam_select(logits.to(dtype).to(DEV), scores.to(DEV), 16))
        order = scores.sort(dim=1, descending=True, stable=True)
        assert torch.equal(s, order.values) and torch.equal(p.long(), order.indices)
        assert torch.equal(t, where[:, :, 0].gather(1, order.indices))
        if V > 500:
            logits = torch.full((1, 8, V), -math.inf)
            for w in range(8):
                logits[0, w, torch.randperm(V, generator=gen)[:40]] = torch.tensor(1.7 * w - 5.3).to(dtype).float()
            s, p, t = (x.cpu() for x in co_alibi_beam_select(logits.to(dtype).to(DEV), torch.zeros(1, 8, device=DEV), 64))
            assert p[0].tolist() == [0] * 40 + [1] * 24 and (s == s[0, 0]).all() and abs(s[0, 0].item() + math.log(40)) < 2.0 ** -21
