"""Logits of both signs of zero are equal: ties go to the lower index."""
import pytest
import torch

from mlperf_training_b200.ops import _lib, moe_ops as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
@pytest.mark.parametrize("groups,top", [(1, 1), (4, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("E,k", [(8, 2), (64, 6), (256, 8)])
def test_zeros_of_both_signs(E, k, dtype, groups, top, score):
    g = torch.Generator().manual_seed(E)
    x = torch.where(torch.rand(500, E, generator=g) < 0.5, -0.0, 0.0)
    x[100:] = torch.where(torch.rand(400, E, generator=g) < 0.1, torch.randn(400, E, generator=g), x[100:])
    x = x.to(dtype)
    got = M.route(x.cuda(), k, score=score, groups=groups, top_groups=top)
    want = M.route(x, k, score=score, groups=groups, top_groups=top)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])
    _lib.check_status("route")
