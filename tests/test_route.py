"""Routing to experts on the CPU: against a token-by-token definition, its gradient against differences, its refusals, and with the experts
behind it."""
import pytest
import torch

from mlperf_training_b200.ops import moe_ops as M
from tests import route_oracle as R

CASES = [
    # T, E, k, score, bias, groups, top_groups, renormalize
    (1, 1, 1, "softmax", False, 1, 1, True),
    (5, 8, 8, "sigmoid", True, 1, 1, True),
    (33, 32, 4, "softmax", False, 1, 1, True),
    (17, 24, 5, "sigmoid", True, 4, 2, True),
    (17, 24, 3, "softmax", True, 8, 3, False),
    (9, 12, 6, "sigmoid", False, 12, 7, False),
    (9, 88, 14, "sigmoid", False, 8, 5, True),
    (3, 256, 32, "softmax", True, 32, 9, True),
]


def inputs(T, E, bias, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * T + E)
    return (torch.randn(T, E, generator=g) * 1.5).to(dtype), 0.2 * torch.randn(E, generator=g) if bias else None


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_route_is_its_definition(case, dtype):
    T, E, k, score, bias, groups, top, renorm = case
    x, b = inputs(T, E, bias, dtype)
    x.requires_grad_(True)
    idx, w, counts = M.route(x, k, score=score, bias=b, groups=groups, top_groups=top, renormalize=renorm, scale=2.5)
    args = (k, score, None if b is None else b.double().tolist(), groups, top, renorm, 2.5)
    want = R.route(x.detach().double().tolist(), *args)
    assert idx.tolist() == want[0] and counts.tolist() == want[2]
    assert idx.dtype == counts.dtype == torch.int32 and w.dtype == torch.float32
    # one rounding to fp32 and the 64-bit arithmetic on both sides
    assert torch.allclose(w.double(), torch.tensor(want[1], dtype=torch.float64), rtol=2 ** -23, atol=1e-30)
    gw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
    dx, = torch.autograd.grad(w, x, gw)
    ref = torch.tensor(R.grad(x.detach().double().tolist(), gw.double().tolist(), *args), dtype=torch.float64)
    assert dx.dtype == dtype
    # one rounding to the logits' type; the rest is what cancels in 64 bits
    assert ((dx.double() - ref).abs() <= ref.abs() * torch.finfo(dtype).eps / 2 * 1.001 + 1e-14).all()


@pytest.mark.parametrize("score,renorm", [("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)])
def test_gradient_against_differences(score, renorm):
    x, b = inputs(3, 12, True)
    x = x.double()
    gw = torch.randn(3, 4, generator=torch.Generator().manual_seed(2)).double()
    args = (4, score, b.double().tolist(), 4, 2, renorm, 1.5)
    ref = torch.tensor(R.grad(x.tolist(), gw.tolist(), *args), dtype=torch.float64)
    h = 1e-6

    def loss(rows):
        return sum(g * v for gr, wr in zip(gw.tolist(), R.route(rows, *args)[1]) for g, v in zip(gr, wr))

    for t in range(3):
        for e in range(12):
            up, down = x.clone(), x.clone()
            up[t, e] += h
            down[t, e] -= h
            # (central differences: third derivatives times h^2 / 6, and 64-bit rounding over h)
            assert abs((loss(up.tolist()) - loss(down.tolist())) / (2 * h) - float(ref[t, e])) < 1e-8


def test_ties_go_to_the_lower_index():
    x = torch.zeros(2, 16)
    x[1, 5] = x[1, 9] = 1.0
    for kw in ({}, {"bias": torch.zeros(16)}, {"groups": 4, "top_groups": 2}):
        idx, w, counts = M.route(x, 3, score="sigmoid", **kw)
        assert idx[0].tolist() == [0, 1, 2]
        assert idx[1].tolist() == ([5, 9, 4] if "groups" in kw else [5, 9, 0])
        assert torch.allclose(w[0], torch.full((3,), 1 / 3))
        assert int(counts.sum()) == 6


def test_infinite_and_not_a_number():
    inf, nan = float("inf"), float("nan")
    # an expert that the bias takes out, one whose logit is masked
    idx, w, _ = M.route(torch.tensor([[3.0, 2.0, -inf, 1.0]]), 2, score="softmax", bias=torch.tensor([-inf, 0, 0, 0]))
    assert idx.tolist() == [[1, 3]] and torch.isfinite(w).all()
    # fewer live experts than k: the masked ones follow by index, with weight 0
    idx, w, _ = M.route(torch.tensor([[-inf, 2.0, -inf, -inf]]), 3)
    assert idx.tolist() == [[1, 0, 2]] and w.tolist() == [[1.0, 0.0, 0.0]]
    # nothing live
    for score in M.ROUTE_SCORES:
        idx, w, _ = M.route(torch.full((1, 4), -inf), 2, score=score)
        assert idx.tolist() == [[0, 1]] and w.tolist() == [[0.0, 0.0]]
    # NaN counts as -inf
    idx, _, _ = M.route(torch.tensor([[nan, -inf, 1.0]]), 3, score="sigmoid")
    assert idx.tolist() == [[2, 0, 1]]


def test_bias_step():
    bias, counts = torch.tensor([0.5, -0.25, 0.0, 1.0]), torch.tensor([4, 0, 2, 2], dtype=torch.int32)
    out = M.balance_bias(bias, counts, 0.125)
    assert out.tolist() == [0.375, -0.125, 0.0, 1.0] and bias[0] == 0.5
    assert M.balance_bias(bias, counts, 0.125, out=bias) is bias and torch.equal(bias, out)


@pytest.mark.parametrize("kw,match", [
    (dict(k=0), "k = 0"), (dict(k=17), "k = 17"), (dict(score="relu"), "relu"), (dict(groups=3), "groups"), (dict(groups=4, top_groups=5), "stay"),
    (dict(groups=4, top_groups=1, k=5), "stay"), (dict(groups=4, top_groups=0), "stay"), (dict(bias=torch.zeros(15)), "bias"),
    (dict(bias=torch.zeros(16, device="meta")), "bias"),
])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        M.route(torch.zeros(2, 16), **{"k": 2, **kw})


@pytest.mark.parametrize("logits", [torch.zeros(16), torch.zeros(2, 16, dtype=torch.float16), torch.zeros(2, 16, dtype=torch.int32), torch.zeros(2, 257)])
def test_refuses_other_logits(logits):
    with pytest.raises(ValueError):
        M.route(logits, 2)


def test_bias_step_refusals():
    with pytest.raises(ValueError):
        M.balance_bias(torch.zeros(4), torch.zeros(5, dtype=torch.int32), 0.1)
    with pytest.raises(ValueError):
        M.balance_bias(torch.zeros(4), torch.zeros(4), 0.1)
    with pytest.raises(ValueError):
        M.balance_bias(torch.zeros(4, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32), 0.1)


def test_no_tokens():
    x = torch.zeros(0, 8, requires_grad=True)
    idx, w, counts = M.route(x, 2)
    w.sum().backward()
    assert idx.shape == w.shape == (0, 2) and counts.tolist() == [0] * 8 and x.grad.shape == (0, 8)


def test_same_as_the_first_router():
    x, _ = inputs(50, 32, False)
    idx, w, counts = M.route(x, 4)
    old = M.router_topk(x, 4)
    assert torch.equal(idx, old[0]) and torch.equal(counts, old[2]) and torch.allclose(w, old[1], rtol=1e-6)


def test_experts_behind_it():
    """Router and experts as a block runs them: output and gradients against autograd in 64 bits."""
    T, D, Fh, E, k = 40, 16, 24, 8, 3
    g = torch.Generator().manual_seed(4)
    h = torch.randn(T, D, generator=g, requires_grad=True)
    logits = torch.randn(T, E, generator=g, requires_grad=True)
    w1 = (torch.randn(E, 2 * Fh, D, generator=g) * 0.2).requires_grad_(True)
    w2 = (torch.randn(E, D, Fh, generator=g) * 0.2).requires_grad_(True)
    bias = 0.3 * torch.randn(E, generator=g)
    idx, w, counts = M.route(logits, k, score="sigmoid", bias=bias, groups=4, top_groups=2, scale=1.5)
    y = M.moe_experts(h, idx, w, counts, w1, w2, residual=h)
    dy = torch.randn(T, D, generator=g)
    got = torch.autograd.grad(y, [h, logits, w1, w2], dy)
    hd, ld, w1d, w2d = (t.detach().double().requires_grad_(True) for t in (h, logits, w1, w2))
    s = torch.sigmoid(ld).gather(1, idx.long())
    wd = 1.5 * s / (s.sum(1, keepdim=True) + 1e-20)
    rows = []
    for t in range(T):
        out = hd[t]
        for j in range(k):
            e = int(idx[t, j])
            gu = w1d[e] @ hd[t]
            out = out + wd[t, j] * (w2d[e] @ (torch.nn.functional.silu(gu[:Fh]) * gu[Fh:]))
        rows.append(out)
    ref = torch.stack(rows)
    want = torch.autograd.grad(ref, [hd, ld, w1d, w2d], dy.double())
    # fp32 products of at most 120 terms on the way: 120 x 2^-24 relative to what is summed, which cancels by less than 10
    for a, b in zip((y,) + got, (ref,) + want):
        assert (a.double() - b).norm() <= 1e-4 * b.norm()
