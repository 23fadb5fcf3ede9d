"""Vocabularies whose marks, with what a block keeps beside them, are about as large as the shared memory that a launch has without asking."""
import pytest
import torch

from mlperf_training_b200.ops import kernels as K
from tests.test_distill import CONFIGS, inputs
from tests.test_gpu_distill import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [CONFIGS[5], CONFIGS[6]], ids=str)
@pytest.mark.parametrize("V", [194000, 195200, 196000, 196576, 196608, 196609, 197000, K.DISTILL_MAX_REST_V])
def test_marks_at_the_limit(V, cfg):
    z, labels, ids, val, gy = inputs(2, V, 9, True, torch.bfloat16)
    check(z, labels, ids, val, gy, cfg)
