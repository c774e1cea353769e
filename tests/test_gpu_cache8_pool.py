"""co_alibi_cache_read_8bit of a pool without pages: every filled row lies on a page outside it.  Needs an MI355X."""
import pytest
import torch

from co_alibi_attn import co_alibi_cache_read_8bit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=str)
@pytest.mark.parametrize("fmt", (torch.float8_e4m3fn, torch.int8), ids=("e4m3", "int8"))
def test_rows_of_a_pool_without_pages(fmt, dtype):
    cache, scale = torch.zeros(0, 2, 16, 64, device=DEV).to(fmt), torch.zeros(0, 2, 1, device=DEV)
    table, lens = torch.zeros(5, 3, dtype=torch.int32, device=DEV), torch.tensor([0, 7, 1000, -3, 20], dtype=torch.int32, device=DEV)
    first = torch.tensor([0, 2, 40, 0, -4], dtype=torch.int32, device=DEV)
    for start in (None, first, first.long()):
        k, v = co_alibi_cache_read_8bit(cache, cache, scale, scale, lens, 60, dtype, table, start)
        row = torch.arange(60, device=DEV) + (0 if start is None else start[:, None].int())
        filled = ((row >= 0) & (row < lens.clamp(max=48)[:, None])).expand(5, 60)
        for x in (k, v):
            assert x.shape == (5, 2, 60, 64) and x.dtype == dtype
            rows = x.transpose(1, 2)
            assert torch.isnan(rows[filled]).all() and (rows[~filled] == 0).all()
