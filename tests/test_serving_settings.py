"""Settings of co_alibi_sample that the host can check."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import co_alibi_attn as co


def test_top_k_is_a_whole_number():
    """0.5 would have been taken as 0, which keeps all."""
    with FakeTensorMode():
        x, u = torch.empty(2, 9, device="cuda"), torch.empty(2, device="cuda")
        for k in (0.5, 1.5, 1e-9, math.nan, -math.inf):
            with pytest.raises(ValueError, match="top_k must be"):
                co.co_alibi_sample(x, u, top_k=k)
        for k in (0, 3, 3.0, 1 << 60, math.inf, True):
            assert co.co_alibi_sample(x, u, top_k=k).shape == (2,)
