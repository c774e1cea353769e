"""8-bit caches that require gradients (float8 tensors can): appends, which write in place, refuse them; reads and decodes keep no record."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import co_alibi_attn as co

E4M3 = torch.float8_e4m3fn


def calls(device, refused):
    """An append of four rows to a cache, one of whose tensors requires gradients, and then a read and a decode over it."""
    on = dict(device=device)
    for which in range(4):
        k = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, **on)
        state = [torch.zeros(2, 2, 32, 64, **on).to(E4M3) for _ in range(2)] + [torch.ones(2, 2, 2, **on) for _ in range(2)]
        state[which].requires_grad_()
        lens = torch.zeros(2, dtype=torch.int32, **on)
        with pytest.raises(ValueError, match="cannot require gradients"):
            co.co_alibi_cache_append_8bit(k, k, *state, lens)
        refused.append(which)
        outs = [*co.co_alibi_cache_read_8bit(*state, lens, 5), co.co_alibi_decode_tree_8bit(k, k, k, *state, seq_len=lens)]
        assert not any(o.requires_grad for o in outs)


def test_without_a_gpu():
    refused = []
    with FakeTensorMode():
        calls("cuda", refused)
    assert refused == [0, 1, 2, 3]


@pytest.mark.gpu
def test_on_the_gpu():
    refused = []
    calls("cuda", refused)
    assert refused == [0, 1, 2, 3]
