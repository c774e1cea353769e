"""co_alibi_decode_tree_8bit over a cache with a NaN in a filled key: the heads that see it get NaN, however far it lies.  Needs an MI355X.

The batch is large enough for a wavefront to walk hundreds of keys, of which steep heads leave the far ones out.
"""
import pytest
import torch

from tests.test_gpu_tree8 import BF16, E4M3, F16, F32, make, run

pytestmark = pytest.mark.gpu

WHERE = (0, 5, 31, 32, 300, 700, 1490, 16, 15, 3, 64)  # one sequence each; those in the oldest tile have nothing behind them


@pytest.mark.parametrize("dtype", (BF16, F16, F32), ids=str)
@pytest.mark.parametrize("T", (1, 3))
@pytest.mark.parametrize("B,n", [(32, 3000), (128, 1500), (200, 1601)])  # from two splits a sequence, whose merge sees all, to one
def test_a_nan_key_reaches_every_row_of_its_head(B, n, T, dtype):
    lens = [n] * B
    q, k, v, caches, scales, table = make(B, 8, 4, T, lens, 16, dtype, E4M3, 16, seed=T)
    want, want_lse = run(q, k, v, caches, scales, table, lens, None)
    assert torch.isfinite(want).all()
    for head in (0, 3):
        bad = caches[0].clone()
        for b, at in enumerate(WHERE):
            bad.view(torch.uint8)[int(table[b, at // 16]), head, at % 16, 9] = 0x7f
        o, lse = run(q, k, v, (bad, caches[1]), scales, table, lens, None)
        hit = torch.zeros(B, 8, dtype=torch.bool)
        hit[:len(WHERE), 2 * head:2 * head + 2] = True
        assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(o[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])
