"""Routing where two groups or two experts lie closer together than the kernel's fp32 values tell apart, against the CPU's 64 bits."""
import pytest
import torch

from mlperf_training_b200.ops import _lib, moe_ops as M

pytestmark = pytest.mark.gpu


def same(x, k, bias=None, **kw):
    got = M.route(x.cuda(), k, bias=None if bias is None else bias.cuda(), **kw)
    want = M.route(x, k, bias=bias, **kw)
    wrong = (got[0].cpu() != want[0]).any(1)
    assert not wrong.any(), f"{int(wrong.sum())} of {len(x)} tokens, the first {int(wrong.nonzero()[0])}"
    assert torch.equal(got[2].cpu(), want[2])
    _lib.check_status("route")


def tied_groups(T, E, G, span, seed=0):
    """Sigmoid logits of which, in each token, the two best of groups 2 and 3 sum up to the same but for a few units of the kernel's fixed point, and biases
    from -span / 2 (in group 1) to span / 2 (in group 0, which therefore stays)."""
    g = torch.Generator().manual_seed(seed + E + G)
    n = E // G
    x = torch.randn(T, E, generator=g).double() - 4.0
    s = 0.3 + 0.6 * torch.rand(T, 3, generator=g).double()
    unit = (1 + span) * 2.0 ** -22
    last = s[:, 0] + s[:, 1] - s[:, 2] + unit * (2 * torch.rand(T, generator=g).double() - 1) * 2
    ok = (last > 0.05) & (last < 0.95)
    last = torch.where(ok, last, 0.5)
    first = 2 * n + torch.randint(0, n - 1, (T,), generator=g)
    for e, v in ((first, s[:, 0]), (first + 1, s[:, 1]), (first + n, s[:, 2]), (first + n + 1, last)):
        x[torch.arange(T), e] = torch.logit(v)
    bias = torch.zeros(E)
    bias[0], bias[n] = span / 2, -span / 2
    return x.float(), bias


@pytest.mark.parametrize("span", [0.5, 3.0, 6.0, 7.0, 8.0, 20.0, 100.0, 1000.0])
@pytest.mark.parametrize("E,G", [(64, 8), (256, 8), (128, 4), (96, 4), (60, 5)])
def test_groups_that_nearly_tie(E, G, span):
    x, bias = tied_groups(20000, E, G, span)
    same(x, 4, bias, score="sigmoid", groups=G, top_groups=2 if span > 4 else 1)


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
def test_groups_that_nearly_tie_without_a_bias(score):
    x, _ = tied_groups(20000, 64, 8, 0.0)
    same(x, 4, score=score, groups=8, top_groups=1)
