"""Infinite biases among groups: a group whose second best expert is switched off is worth -inf, one with an expert switched on +inf."""
import pytest
import torch

from mlperf_training_b200.ops import _lib, moe_ops as M
from tests.test_route_switched_off import CASES, switched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["off", "on", "both"])
@pytest.mark.parametrize("E,G,top,k", CASES + [(256, 8, 4, 8), (96, 32, 10, 5), (160, 20, 7, 32)])
def test_groups_with_infinite_biases(E, G, top, k, kind, dtype, score):
    x, bias = switched(600, E, G, kind)
    x = x.to(dtype)
    got = M.route(x.cuda(), k, score=score, bias=bias.cuda(), groups=G, top_groups=top)
    want = M.route(x, k, score=score, bias=bias, groups=G, top_groups=top)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])
    assert torch.allclose(got[1].cpu(), want[1], rtol=2e-6, atol=1e-30)
    _lib.check_status("route")
