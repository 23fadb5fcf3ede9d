"""Numbers of tokens and of logits that the kernels' 32-bit counters do not hold are refused."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K


@pytest.mark.parametrize("T", [K.DISTILL_MAX_T + 1, 2 ** 31 - 1, 2 ** 32 + 5])
def test_too_many_tokens(T):
    z, ids, val = torch.zeros(1, 2).expand(T, 2), torch.zeros(1, 1, dtype=torch.int32).expand(T, 1), torch.zeros(1, 1).expand(T, 1)
    with pytest.raises(ValueError, match="tokens"):
        F.distill_loss(z, None, ids, val)


@pytest.mark.parametrize("V", [K.DISTILL_MAX_V + 1, 2 ** 32 + 5])
def test_too_many_logits(V):
    with pytest.raises(ValueError, match="logits"):
        F.distill_loss(torch.zeros(1, 1, dtype=torch.bfloat16).expand(1, V), None, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1))


def test_row_counters_stay_in_32_bits():
    # a block goes on by a grid's worth of rows at a time: 10 blocks to an SM
    assert K.DISTILL_MAX_T + 10 * 1000 < 2 ** 31
