"""Caches of no rows: a block table without blocks, as before the first page of a batch is given out.  Needs an MI355X."""
import pytest
import torch

from co_alibi_attn import co_alibi_cache_append, co_alibi_decode_tree

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=str)
def test_a_table_without_blocks(dtype):
    gen = torch.Generator(device=DEV).manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)  # noqa: E731
    q, k, v, kc, vc = n(2, 4, 3, 64), n(2, 2, 3, 64), n(2, 2, 3, 64), n(5, 2, 16, 64), n(5, 2, 16, 64)
    table = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    some = torch.tensor([[0], [3]], dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    want = co_alibi_decode_tree(q, k, v, kc, vc, seq_len=lens, block_table=some)
    for kw in (dict(), dict(seq_len=0), dict(seq_len=lens), dict(seq_len=lens + 9)):
        assert torch.equal(co_alibi_decode_tree(q, k, v, kc, vc, block_table=table, **kw), want)
        assert torch.equal(co_alibi_decode_tree(q, k, v, kc[:0], vc[:0], block_table=table, **kw), want)
    before = kc.clone(), vc.clone()
    co_alibi_cache_append(k, v, kc, vc, lens, block_table=table)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
