"""Routing kernels against the same operator on the CPU, which computes in 64 bits (and is held to the definition by its own tests)."""
import pytest
import torch

from mlperf_training_b200.ops import _lib, moe_ops as M
from tests.test_route import CASES, inputs

pytestmark = pytest.mark.gpu

MORE = [(T, E, k, score, bias, groups, top, renorm)
        for T, E, k in ((1, 33, 3), (7, 64, 6), (8, 128, 8), (9, 130, 2), (1000, 255, 7), (20011, 96, 4))
        for score, bias, groups, top, renorm in (("softmax", False, 1, 1, True), ("sigmoid", True, 1, 1, False), ("softmax", True, 1, 1, True))]
MORE += [(4099, 64, 6, "sigmoid", True, 8, 4, True), (3001, 256, 8, "sigmoid", True, 8, 4, True), (513, 96, 5, "softmax", False, 32, 10, False),
         (77, 60, 9, "sigmoid", True, 5, 3, True), (600, 31, 31, "softmax", False, 31, 31, False), (40, 160, 32, "sigmoid", True, 20, 7, True)]


def check(x, b, gw, k, kw):
    xg = x.cuda().requires_grad_(True)
    idx, w, counts = M.route(xg, k, bias=None if b is None else b.cuda(), **kw)
    dx, = torch.autograd.grad(w, xg, gw.cuda())
    want = M.route(x, k, bias=b, **kw)
    # (in 64 bits: a reference rounded to the logits' type would lie on the other side of a tie now and then)
    ref = M.route_bwd(gw, x.double(), want[0], score=kw["score"], renormalize=kw.get("renormalize", True), scale=kw.get("scale", 1.0))
    assert torch.equal(idx.cpu(), want[0]) and torch.equal(counts.cpu(), want[2])
    # a score in fp32: exponential 2^-22 + |x| 2^-24 (|x| < 9), reciprocal 2^-23, sum of k and quotient 2^-22; below 1e-6 together
    assert torch.allclose(w.cpu(), want[1], rtol=2e-6, atol=1e-30)
    # dL/ds: two such quotients of sums whose terms cancel; then the rounding to the logits' type
    size = kw.get("scale", 1.0) * gw.abs().amax(1, keepdim=True)
    if kw.get("renormalize", True):
        s = M._route_scores(x.double(), kw["score"]).gather(1, want[0].long())
        size = size / (s.sum(1, keepdim=True) + M.ROUTE_EPS).float()
    s = M._route_scores(x.double(), kw["score"]).float()
    bound = torch.finfo(x.dtype).eps / 2 * 1.01 * ref.abs() + 6e-6 * size * s + 1e-30
    assert ((dx.cpu().double() - ref).abs() <= bound + torch.finfo(x.dtype).eps / 2 * bound).all()
    _lib.check_status("route")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES + MORE, ids=str)
def test_route(case, dtype):
    T, E, k, score, bias, groups, top, renorm = case
    x, b = inputs(T, E, bias, dtype)
    gw = torch.randn(T, k, generator=torch.Generator().manual_seed(1))
    check(x, b, gw, k, dict(score=score, groups=groups, top_groups=top, renormalize=renorm, scale=2.5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("E,off,pitch", [(64, 1, 67), (64, 8, 72), (96, 3, 99), (256, 4, 260)])
def test_rows_of_a_wider_buffer(E, off, pitch, dtype):
    """Rows that are not aligned, or further apart than they are long."""
    buf = torch.randn(50, pitch, generator=torch.Generator().manual_seed(E + off)).to(dtype)
    x = buf[:, off:off + E]
    got = M.route(buf.cuda()[:, off:off + E], 5, score="sigmoid", groups=4, top_groups=2)
    for a, b in zip(got, M.route(x, 5, score="sigmoid", groups=4, top_groups=2)):
        assert torch.equal(a.cpu(), b) if a.dtype == torch.int32 else torch.allclose(a.cpu(), b, rtol=2e-6)
    t = M.route(buf.t().contiguous().t().cuda()[:, off:off + E], 5, score="sigmoid", groups=4, top_groups=2)     # columns apart
    assert torch.equal(t[0], got[0])
    _lib.check_status("route")


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
@pytest.mark.parametrize("groups,top", [(1, 1), (8, 4)])
def test_choices_that_fp32_does_not_resolve(score, groups, top):
    """Scores plus biases that all lie within a few 1e-8 of one value, in another order in fp32 than in 64 bits."""
    T, E, k = 64, 64, 6
    x = torch.randn(1, E, generator=torch.Generator().manual_seed(5)).expand(T, E).contiguous()
    x = x + 0.0 * torch.arange(T)[:, None]
    s = M._route_scores(x[:1].double(), score)[0]
    b = (0.75 - s).float()
    assert ((s + b.double()) - 0.75).abs().max() < 1e-7
    got = M.route(x.cuda(), k, score=score, bias=b.cuda(), groups=groups, top_groups=top)
    want = M.route(x, k, score=score, bias=b, groups=groups, top_groups=top)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])


def test_infinite_and_not_a_number():
    inf, nan = float("inf"), float("nan")
    x = torch.randn(40, 48, generator=torch.Generator().manual_seed(6))
    x[0] = -inf
    x[1, 1:] = -inf
    x[2, ::2] = -inf
    x[3, 7] = nan
    x[4, :40] = nan
    b = torch.zeros(48)
    b[5], b[11] = -inf, 3.0
    for score in M.ROUTE_SCORES:
        for kw in ({}, {"bias": b}, {"bias": b, "groups": 6, "top_groups": 3}):
            got = M.route(x.cuda(), 4, score=score, **{n: v.cuda() if torch.is_tensor(v) else v for n, v in kw.items()})
            want = M.route(x, 4, score=score, **kw)
            same = torch.ones(40, dtype=torch.bool)
            if score == "softmax" and kw:
                same[3:5] = False                  # (a softmax over NaN is all NaN: any choice in range)
            assert torch.equal(got[0].cpu()[same], want[0][same])
            assert torch.allclose(got[1].cpu()[same], want[1][same], rtol=2e-6, equal_nan=True)
            assert int(got[0].min()) >= 0 and int(got[0].max()) < 48
    _lib.check_status("route")


def test_repeats_are_equal_and_streams_are_kept():
    x, b = inputs(30000, 64, True)
    x, b = x.cuda(), b.cuda()
    first = M.route(x, 6, score="sigmoid", bias=b, groups=8, top_groups=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = M.route(x, 6, score="sigmoid", bias=b, groups=8, top_groups=4)
        bias = M.balance_bias(b, again[2], 1e-3)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    assert torch.equal(bias.cpu(), M.balance_bias(b.cpu(), first[2].cpu(), 1e-3))


def test_captured_and_replayed():
    x, b = inputs(300, 64, True)
    x, b = x.cuda(), b.cuda()
    M.route(x, 6, score="sigmoid", bias=b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = M.route(x, 6, score="sigmoid", bias=b)
        nb = M.balance_bias(b, out[2], 1e-3)
    for seed in (1, 2):
        x.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = M.route(x, 6, score="sigmoid", bias=b)
        assert all(torch.equal(p, q) for p, q in zip(out, want)) and torch.equal(nb, M.balance_bias(b, want[2], 1e-3))
    _lib.check_status("route")


def test_experts_behind_it():
    """Router, plan and experts as a block runs them, on the GPU's kernels against the CPU's bodies."""
    T, D, Fh, E, k = 333, 128, 192, 16, 4
    g = torch.Generator().manual_seed(4)
    h = torch.randn(T, D, generator=g).bfloat16()
    logits = torch.randn(T, E, generator=g)
    w1, w2 = ((torch.randn(E, *s, generator=g) * 0.1).bfloat16() for s in ((2 * Fh, D), (D, Fh)))
    bias, dy = 0.3 * torch.randn(E, generator=g), torch.randn(T, D, generator=g).bfloat16()
    out = []
    for dev in ("cpu", "cuda"):
        v = [t.to(dev).requires_grad_(True) for t in (h, logits, w1, w2)]
        idx, w, counts = M.route(v[1], k, score="sigmoid", bias=bias.to(dev), groups=4, top_groups=2, scale=1.5)
        y = M.moe_experts(v[0], idx, w, counts, v[2], v[3], residual=v[0])
        out.append([t.detach().float().cpu() for t in (y, *torch.autograd.grad(y, v, dy.to(dev)))])
    # bf16 in the same places on both sides (rounded from sums in another order: a flip is 2^-8 of an element, and four such steps follow
    # one another on the way to each result)
    for a, b in zip(*out):
        assert (a - b).norm() <= 4 * 2 ** -8 * b.norm()
    _lib.check_status("route")
