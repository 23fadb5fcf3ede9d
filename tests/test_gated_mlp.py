"""Gated feed-forward block on the CPU: against 64 bits, gradients against autograd of the formula and differences, refusals."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K

ACT = {"silu": torch.nn.functional.silu, "gelu": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}


def plain(x, w_gu, w_down, r, act):
    g, u = (x @ w_gu.t()).chunk(2, 1)
    y = (ACT[act](g) * u) @ w_down.t()
    return y if r is None else y + r


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,D,Fh,Do", [(1, 8, 8, 8), (7, 24, 40, 16)])
def test_gradients_are_the_formulas(act, T, D, Fh, Do):
    torch.manual_seed(T)
    t = [torch.randn(*s).requires_grad_() for s in ((T, D), (2 * Fh, D), (Do, Fh), (T, Do))]
    d = [v.detach().double().requires_grad_() for v in t]
    y, yd = F.gated_mlp(*t, act=act), plain(*d, act)
    assert torch.allclose(y.double(), yd, atol=1e-5 * float(yd.detach().abs().max()))
    dy = torch.randn(T, Do)
    for a, b in zip(torch.autograd.grad(y, t, dy), torch.autograd.grad(yd, d, dy.double())):
        assert torch.allclose(a.double(), b, atol=1e-5 * float(b.abs().max()))
    v = [torch.randn_like(a) for a in d]
    f = lambda e: (plain(*[a.detach() + e * b for a, b in zip(d, v)], act) * dy.double()).sum()
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(float(sum((g.double() * b).sum() for g, b in zip(torch.autograd.grad(F.gated_mlp(*t, act=act), t, dy), v)) / slope) - 1) < 1e-4


def test_main_grad_no_grad_and_no_tokens():
    torch.manual_seed(0)
    x, w1, w2 = torch.randn(4, 8, requires_grad=True), torch.nn.Parameter(torch.randn(32, 8)), torch.nn.Parameter(torch.randn(8, 16))
    want = torch.autograd.grad(F.gated_mlp(x, w1, w2).sum(), [w1, w2])
    w1.main_grad, w2.main_grad = torch.zeros(32, 8), torch.zeros(8, 16)
    F.gated_mlp(x, w1, w2).sum().backward()
    assert w1.grad is None and torch.allclose(w1.main_grad, want[0], atol=1e-5) and torch.allclose(w2.main_grad, want[1], atol=1e-5)
    with torch.no_grad():
        assert not F.gated_mlp(x, w1, w2).requires_grad
    e = torch.zeros(0, 8, requires_grad=True)
    y = F.gated_mlp(e, torch.nn.Parameter(torch.randn(32, 8)), torch.nn.Parameter(torch.randn(8, 16)))
    y.sum().backward()
    assert y.shape == (0, 8) and e.grad.shape == (0, 8)


def test_refusals():
    x, w1, w2 = torch.randn(4, 8), torch.randn(32, 8), torch.randn(8, 16)
    for bad in (lambda: F.gated_mlp(x, w1, torch.randn(8, 15)), lambda: F.gated_mlp(x, torch.randn(32, 9), w2),
                lambda: F.gated_mlp(x, w1, w2, residual=torch.randn(4, 9)), lambda: F.gated_mlp(x, w1, w2, act="relu"),
                lambda: F.gated_mlp(torch.randn(8), w1, w2), lambda: K.gated_fwd(x, torch.randn(31, 8)),
                lambda: K.gated_bwd(x, w2, torch.randn(4, 30))):
        with pytest.raises(ValueError):
            bad()
