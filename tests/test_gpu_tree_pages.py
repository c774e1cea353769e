"""Block-table entries outside the pool, at every place of a chunk of keys: every row of the sequence is NaN, in each
form of co_alibi_decode_tree (row blocks of 32, 64 and 128, whole sequences and splits).  Needs an MI355X.

The entries are caught on the device: such a page's rows are read from page 0, inside the pool.
"""
import pytest
import torch

from co_alibi_attn import co_alibi_decode_tree

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HKV, G, D = 2, 4, 128


def inputs(B, T, L, page, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(torch.bfloat16)  # noqa: E731
    blocks = -(-L // page)
    q, k, v = n(B, G * HKV, T, D), n(B, HKV, T, D), n(B, HKV, T, D)
    pools = n(B * blocks, HKV, page, D), n(B * blocks, HKV, page, D)
    table = torch.randperm(B * blocks, generator=gen, device=DEV).view(B, blocks).to(torch.int32)
    return q, k, v, *pools, table


def run(q, k, v, kc, vc, table, seq_len):
    out = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=seq_len, block_table=table, return_lse=True)
    torch.cuda.synchronize()
    return out


def check(got, sound, bad):
    for x, y in zip(got, sound):
        for b in range(x.shape[0]):
            if b in bad:
                assert x[b].isnan().all(), (b, int(x[b].isnan().sum()), x[b].numel())
            else:
                assert torch.equal(x[b], y[b]), b


@pytest.mark.parametrize("page", (16, 32, 64, 128))
@pytest.mark.parametrize("T", (1, 8, 9, 16, 17, 32, 33), ids=lambda t: f"rows{G * t}")
def test_few_sequences_over_many_splits(T, page):
    B, L = 3, 3000
    args = inputs(B, T, L, page, seed=T)
    sound = run(*args, L)
    blocks = args[5].shape[1]
    # The oldest 256 rows (every place of two chunks), one in the middle, and the newest, partly filled ones.
    for place in sorted({*range(256 // page), blocks // 2, blocks - 2, blocks - 1}):
        table = args[5].clone()
        table[1, place] = args[3].shape[0] if place % 2 else -1
        print(T, page, place, flush=True)
        check(run(*args[:5], table, L), sound, {1})


@pytest.mark.parametrize("page", (16, 32, 64))
@pytest.mark.parametrize("T", (1, 9, 16, 17, 33), ids=lambda t: f"rows{G * t}")
def test_many_sequences_one_work_group_each(T, page):
    """So many that each goes through one work-group, without a merge; every odd one has a bad entry of its own."""
    B, L = 300, 200
    args = inputs(B, T, L, page, seed=100 + T)
    sound = run(*args, L)
    table, blocks = args[5].clone(), args[5].shape[1]
    odd = range(1, B, 2)
    for b in odd:
        table[b, b // 2 % blocks] = -1 - b
    check(run(*args[:5], table, L), sound, set(odd))


@pytest.mark.parametrize("T", (1, 16, 17), ids=lambda t: f"rows{G * t}")
def test_ragged_batch(T):
    """Splits shared out by the sequences' own lengths; entries past a sequence's filled rows are never looked at."""
    B, page, lens = 24, 16, [0, 1, 5, 16, 17, 40, 63, 64, 65, 90, 127, 128, 129, 130, 192, 200, 255, 256, 300, 512, 700, 2900, 1500, 77]
    args = inputs(B, T, max(lens), page, seed=200 + T)
    seq_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    sound = run(*args, seq_len)
    for step in range(4):
        table, bad = args[5].clone(), set()
        for b, n in enumerate(lens):
            filled = -(-n // page)
            table[b, filled:] = -9
            if b % 4 == step and filled:
                table[b, (5 * b + step) % filled] = 1 << 30
                bad.add(b)
        check(run(*args[:5], table, seq_len), sound, bad)
