"""co_alibi_decode_tree_8bit with fp16 inputs over blocks of V whose scales lie far apart.  Needs an MI355X.

Channels in which the blocks of large scales hold zeros are sums of the small blocks' values alone: weights of 11 bits each, as
over a cache of fp16 values.  All codes are >= 0 there, so that o is its own sum of sizes: an error of e in each weight
and in the sum is 2 e o, and the output's rounding e o (2^-25 below fp16's normal numbers), with e = 2^-11.  Weights below 2^-14 of the
row's largest, which the sum is not below, have errors of up to 2^-25 of it: 2^-25 of the sum of the row's values.
"""
import pytest
import torch

from oracle import serving8 as oracle
from tests.test_gpu_tree8 import F16, FORMATS, make, run, slopes, within

pytestmark = pytest.mark.gpu


def small_channels(lens, D, fmt, T, seed, ratio, order):
    q, k, v, caches, scales, table = make(len(lens), 4, 2, T, lens, D, F16, fmt, 16, seed=seed)
    half = D // 2
    gen = torch.Generator().manual_seed(seed)
    code = lambda *s: torch.randint(1, 100, s, generator=gen).double()  # noqa: E731
    vc, vs = caches[1].double(), scales[1].clone()
    for b, n in enumerate(lens):
        for j in range(-(-n // 16)):
            u, rows = int(table[b, j]), min(16, n - 16 * j)
            large = order(j)
            vs[u] = 2.0 ** 6 if large else 2.0 ** 6 * ratio
            vc[u, :, :rows] = code(vc.shape[1], rows, D)
            if large:
                vc[u, :, :rows, half:] = 0
    v = v.abs()
    v[..., half:] = 0
    return q, k, v, (caches[0], oracle.code(vc, fmt).to(fmt)), (scales[0], vs), table


@FORMATS
@pytest.mark.parametrize("ratio", (2.0 ** -10, 2.0 ** -14, 2.0 ** -16, 2.0 ** -18, 2.0 ** -14 * 1.3))
def test_small_values_beside_large_ones(ratio, fmt):
    for lens, D, T, order in (([40, 16], 64, 1, lambda j: j % 2), ([300, 170], 32, 5, lambda j: j % 3 != 1), ([700], 128, 3, lambda j: j < 20),
                              ([700], 16, 2, lambda j: j > 20), ([90, 500], 256, 1, lambda j: j % 4 == 0)):
        args = small_channels(lens, D, fmt, T, D, ratio, order)
        q, k, v, caches, scales, table = args
        o, _ = run(*args, lens, None)
        want, _, ob, _ = oracle.decode_tree(q.float(), k.float(), v.float(), caches, scales, lens, None, table, slopes(4, 8.0, F16),
                                            D ** -0.5)
        vals = oracle.values(caches[1], scales[1])
        sizes = torch.stack([oracle.rows_of(vals, table, b, 0, n).abs().sum(1) for b, n in enumerate(lens)]) + v.double().sum(2)
        rare = 2.0 ** -25 * (1 + sizes.repeat_interleave(2, 1)[:, :, None])
        over = (o.double() - want).abs() - (ob + 3.1 * 2.0 ** -11 * want.abs() + rare)
        assert over.max() <= 0, (lens, D, float(over.max()), int((over > 0).sum()))


@FORMATS
def test_scales_over_the_whole_range(fmt):
    """Blocks from 2^-40 to as much as fp16's outputs hold, growing and shrinking from key to key, with one or several splits; and
    large scales over codes of zero."""
    for lens, T, step in (([333, 64], 5, 1), ([2500, 31], 1, 7), ([90, 100], 40, 13)):
        q, k, v, caches, scales, table = make(2, 4, 2, T, lens, 64, F16, fmt, 16, seed=9)
        scales = [s.clone() for s in scales]
        for b, n in enumerate(lens):
            for j in range(-(-n // 16)):
                scales[1][int(table[b, j])] = 2.0 ** (-40 + step * j % 46) * (1.0 if j % 3 else 1.4)
        zero = int(table[0, 2])
        caches[1].view(torch.uint8)[zero] = 0
        scales[1][zero] = 2.0 ** 40
        args = q, k, v, caches, scales, table
        o, lse = run(*args, lens, None)
        want = oracle.decode_tree(*args[:3], caches, scales, lens, None, table, slopes(4, 8.0, F16), 0.125)
        within(o, lse, want)
