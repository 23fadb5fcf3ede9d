"""Caps of attention scores whose squares fp32 does not hold are refused."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F


@pytest.mark.parametrize("cap", [1e-45, 1e-13, 1e19, 1e38])
def test_caps_out_of_range(cap):
    q = torch.zeros(1, 3, 2, 8)
    with pytest.raises(ValueError, match="softcap"):
        F.masked_attention(q, q, q, F.attention_mask(1, 3), softcap=cap)


@pytest.mark.parametrize("cap", [1e-12, 1e18])
def test_caps_at_the_ends(cap):
    q = torch.randn(1, 3, 2, 8, generator=torch.Generator().manual_seed(0))
    y = F.masked_attention(q, q, q, F.attention_mask(1, 3), softcap=cap)
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), q.double()) * 8 ** -0.5
    p = torch.softmax((cap * torch.tanh(s / cap)).masked_fill(~torch.ones(3, 3).tril().bool(), -torch.inf), -1)
    assert torch.allclose(y.double(), torch.einsum("bhqk,bkhd->bqhd", p, q.double()), rtol=1e-6, atol=1e-6)
