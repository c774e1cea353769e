"""co_alibi_sample at the ends of fp32's and of the settings' ranges, against the float64 oracle.  Needs an MI355X.

The draws are given by small counts of equal weights or weights far apart, so that no border lies near a uniform number.
"""
import math

import pytest
import torch

from co_alibi_attn import co_alibi_sample
from oracle import serving as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def check(x, u, t=1.0, k=0, p=1.0, m=0.0):
    got = co_alibi_sample(x.to(DEV), u.to(DEV), temperature=t, top_k=k, top_p=p, min_p=m).tolist()
    B = x.shape[0]
    assert got == oracle.sample(x, u, [t] * B, [k] * B, [p] * B, [m] * B), (t, k, p, m)


U = torch.tensor([0.03, 0.2, 0.45, 0.55, 0.8, 0.97])


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_logits_further_apart_than_the_largest_number(dtype):
    """Their distance is no fp32 number; at such temperatures their weights are not 0 all the same."""
    top = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(1)
    few = torch.tensor([top, -top, 0.5 * top, -0.9 * top, 0.0, -math.inf], dtype=dtype).expand(6, 6)
    many = (torch.rand(6, 5000, generator=gen) * 2 - 1).mul(top).to(dtype)
    for x in (few, many):
        for t in (1e37, 1e38, 3e38, 1e39, 1e300, math.inf):
            for kw in (dict(), dict(k=3), dict(k=900), dict(p=0.7), dict(m=0.3)):
                print(x.shape, t, kw, flush=True)
                check(x, U, t=t, **kw)


def test_min_p_and_temperature_both_far_below_fp32():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(6, 5000, generator=gen)
    ties = torch.randint(0, 3, (6, 3000), generator=gen).float()
    wide = x * 1e37
    for rows in (x, ties, wide, x * 1e-42, x.to(torch.bfloat16), x[:, :5]):
        for t in (5e-324, 1e-300, 1e-46, 1e-40, 1e-6, 1.0, 1e300, math.inf):
            for m in (5e-324, 1e-300, 1e-46, 1e-39, 1e-20):
                for p in (1.0, 0.6):
                    print(rows.shape, t, m, p, flush=True)
                    check(rows, U, t=t, m=m, p=p)
