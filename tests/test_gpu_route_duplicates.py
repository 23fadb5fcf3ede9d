"""Experts of equal logits at the border of the choice, with others that differ from them by less than the kernel's keys hold."""
import pytest
import torch

from mlperf_training_b200.ops import _lib, moe_ops as M

pytestmark = pytest.mark.gpu


def resolved(x, score, groups=1, top_groups=1):
    """Tokens whose groups 64 bits tell apart.  A group of two copies d above and d below another's has e^d + e^-d = 2 + d^2 where that has 2, and a
    few units of fp32 make d^2 2^-46 to 2^-60: exponentials and sums in 64 bits are off by a few 2^-53 of a value themselves, and two
    of them give either order.  (A tie in the same bits on both sides, of the same logits, is a tie for any of them.)"""
    if groups == top_groups:
        return torch.ones(len(x), dtype=torch.bool)
    by = x.double().unflatten(1, (groups, -1)).sort(-1, descending=True)[0][..., :2]
    value = M._route_scores(x.double(), score).unflatten(1, (groups, -1)).sort(-1, descending=True)[0][..., :2].sum(-1)
    near = (value[:, :, None] - value[:, None]).abs() <= 16 * 2 ** -53 * value[:, :, None]
    return ~(near & (by[:, :, None] != by[:, None]).any(-1)).any(2).any(1)


def same(x, k, **kw):
    got, want = M.route(x.cuda(), k, **kw), M.route(x, k, **kw)
    at = resolved(x, **kw)
    assert at.float().mean() > 0.9                     # (of the inputs alone: 1 % of them at most)
    assert torch.equal(got[0].cpu()[at], want[0][at]) and int((got[2].cpu() - want[2]).abs().sum()) <= 2 * k * int((~at).sum())
    assert torch.allclose(got[1].cpu()[at], want[1][at], rtol=2e-6, atol=1e-30)
    _lib.check_status("route")


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
def test_a_larger_logit_behind_two_equal_ones(score):
    same(torch.tensor([[1.0, 1.0, 1.0 + 1e-6], [-1.0, -1.0, -1.0 + 1e-6], [1.0, 1.0 + 1e-6, 1.0], [2.0, 2.0, 2.0]]), 1, score=score)


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
@pytest.mark.parametrize("groups,top", [(1, 1), (4, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("E,k", [(8, 2), (32, 4), (64, 6), (96, 7), (256, 8), (256, 32)])
def test_copies_of_experts(E, k, dtype, groups, top, score):
    """Rows of which many are copies, copies a few units up or down, and zeros."""
    T = 4000
    g = torch.Generator().manual_seed(E + k)
    base = torch.randn(T, max(E // 8, 2), generator=g)
    x = base.gather(1, torch.randint(0, base.shape[1], (T, E), generator=g))
    units = torch.randint(-3, 4, (T, E), generator=g) * (torch.rand(T, E, generator=g) < 0.3)
    x = (x.view(torch.int32) + units.int()).view(torch.float32)
    x[::7] = 0.0
    x[1::7, : E // 2] = float("-inf")
    same(x.to(dtype), k, score=score, groups=groups, top_groups=top)
