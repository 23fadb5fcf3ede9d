"""Operators whose autograd nodes are the host module's: the same results as through torch.autograd.Function, and what a node has to keep to
(a second backward pass, changed operands, hooks, other streams, partial gradients)."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import moe_ops as M
from tests.test_masked_attention import documents

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def module():
    if _lib.host is None:
        pytest.skip("the host module is not built")


def randn(*s, seed=0, dtype=torch.float32):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed + sum(s))).to(dtype).cuda()


def route(T=50):
    x, b = randn(T, 64, dtype=torch.bfloat16).requires_grad_(True), 0.1 * randn(64)
    idx, w, counts = M.route(x, 5, score="sigmoid", bias=b, groups=8, top_groups=4, scale=1.5)
    return [idx, w, counts], w, [x], randn(T, 5, seed=1)


def distill(T=50):
    z = randn(T, 999, dtype=torch.bfloat16).requires_grad_(True)
    labels, ids = torch.arange(T).cuda(), (torch.arange(T * 7).view(T, 7) * 13 % 999).cuda()
    loss = F.distill_loss(z, labels, ids, randn(T, 7), alpha=0.6, temperature=2.0)
    return [loss], loss, [z], randn(T, seed=1)


def attention(S=200, **kw):
    q, k, v = (randn(2, S, h, 64, seed=h, dtype=torch.bfloat16).requires_grad_(True) for h in (4, 2, 2))
    y = F.masked_attention(q, k, v, F.attention_mask(2, S, documents=documents(2, S, "few").cuda()), softcap=9.0, slopes=0.1 * torch.ones(4).cuda(), **kw)
    return [y], y, [q, k, v], randn(2, S, 4, 64, seed=1, dtype=torch.bfloat16)


OPS = {"route": route, "distill": distill, "attention": attention}


@pytest.mark.parametrize("name", OPS)
def test_same_as_without_the_module(name, monkeypatch):
    def run():
        out, y, ins, g = OPS[name]()
        return [t.detach() for t in out] + list(torch.autograd.grad(y, ins, g)), type(y.grad_fn).__name__
    a, node = run()
    monkeypatch.setattr(_lib, "host", None)
    b, other = run()
    assert node != other
    for i, (p, q) in enumerate(zip(a, b)):
        if name == "attention" and i == 1:                     # dQ is added up in another order each time
            assert (p.float() - q.float()).norm() <= 2 ** -8 * q.float().norm()
        else:
            assert torch.equal(p, q)
    _lib.check_status(name)


@pytest.mark.parametrize("name", OPS)
def test_node(name):
    out, y, ins, g = OPS[name]()
    seen = []
    ins[0].register_hook(lambda t: seen.append(t.shape))
    first = torch.autograd.grad(y, ins, g, retain_graph=True)
    again = torch.autograd.grad(y, ins[:1], g, retain_graph=True)
    assert seen == [ins[0].shape] * 2
    if name != "attention":
        assert torch.equal(first[0], again[0])
    y.backward(g)
    assert all(t.grad is not None and t.grad.shape == t.shape and t.grad.dtype == t.dtype for t in ins)
    with pytest.raises(RuntimeError, match="second time"):
        y.backward(g)
    # an operand that was changed in place since is noticed
    out, y, ins, g = OPS[name]()
    with torch.no_grad():
        ins[0].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


@pytest.mark.parametrize("name", OPS)
def test_without_gradients(name):
    with torch.no_grad():
        out, y, _, _ = OPS[name]()
    assert y.grad_fn is None and not y.requires_grad
    out, y, ins, g = OPS[name]()
    assert y.requires_grad and all(not t.requires_grad for t in out if t is not y)


@pytest.mark.parametrize("name", OPS)
def test_another_stream_and_gradients_of_other_layouts(name):
    out, y, ins, g = OPS[name]()
    want = torch.autograd.grad(y, ins, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, y, ins, _ = OPS[name]()
        apart = torch.stack([g, g], -1)[..., 0]                # strided
        got = torch.autograd.grad(y, ins, apart)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert (a.float() - b.float()).norm() <= 2 ** -8 * b.float().norm()
    _lib.check_status(name)


def captured_route():
    b = 0.1 * randn(64)
    return [randn(50, 64, dtype=torch.bfloat16)], randn(50, 5, seed=1), lambda x: M.route(x, 5, score="sigmoid", bias=b, groups=8, top_groups=4)[1]


def captured_distill():
    labels, ids, values = torch.arange(50).cuda(), (torch.arange(350).view(50, 7) * 13 % 999).cuda(), randn(50, 7)
    return [randn(50, 999, dtype=torch.bfloat16)], randn(50, seed=1), lambda z: F.distill_loss(z, labels, ids, values, alpha=0.6, temperature=2.0)


def captured_attention():
    ids, slopes = documents(2, 200, "few").cuda(), 0.1 * torch.ones(4).cuda()
    return ([randn(2, 200, h, 64, seed=h, dtype=torch.bfloat16) for h in (4, 2, 2)], randn(2, 200, 4, 64, seed=1, dtype=torch.bfloat16),
            lambda q, k, v: F.masked_attention(q, k, v, F.attention_mask(2, 200, documents=ids), softcap=9.0, slopes=slopes))


@pytest.mark.parametrize("make", [captured_route, captured_distill, captured_attention])
def test_captured_and_replayed_with_its_gradient(make):
    given, g, f = make()
    fed = [t.clone() for t in given]

    def step():
        ins = [t.detach().requires_grad_(True) for t in fed]
        y = f(*ins)
        return [y.detach()] + list(torch.autograd.grad(y, ins, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in (0, 1):
        for t, x in zip(fed, given):
            t.copy_(x.roll(turn, -1))
        graph.replay()
        for a, b in zip(step(), got):                          # (dQ is added up in another order each time)
            assert torch.isfinite(a.float()).all() and (a.float() - b.float()).norm() <= 2 ** -8 * a.float().norm()
    _lib.check_status(make.__name__)


def test_sink_takes_the_general_path():
    sink = torch.zeros(4, device="cuda", requires_grad=True)
    out, y, ins, g = attention(sink=sink)
    assert torch.isfinite(torch.autograd.grad(y, [sink], g)[0]).all()


def test_gradient_of_one_operand_alone():
    q, k = randn(1, 40, 2, 64, dtype=torch.bfloat16), randn(1, 40, 2, 64, seed=3, dtype=torch.bfloat16)
    v = randn(1, 40, 2, 64, seed=4, dtype=torch.bfloat16).requires_grad_(True)
    y = F.masked_attention(q, k, v, F.attention_mask(1, 40, device="cuda"))
    y.sum().backward()
    assert v.grad is not None and torch.isfinite(v.grad.float()).all()


def test_refusals_are_the_general_paths():
    x = torch.zeros(4, 16, device="cuda")
    with pytest.raises(ValueError, match="route"):
        M.route(x, 17)
    with pytest.raises(ValueError, match="route"):
        M.route(x, 2, score="relu")
    with pytest.raises(ValueError, match="distill"):
        F.distill_loss(x, None, torch.zeros(4, 3, dtype=torch.int64).cuda(), torch.zeros(4, 3).cuda(), alpha=0.5)
    with pytest.raises(ValueError, match="distill"):
        F.distill_loss(x, None, torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3).cuda())
    m = F.attention_mask(1, 4, device="cuda")
    b = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(softcap=-1.0), dict(scale=0.0), dict(slopes=torch.zeros(3).cuda())):
        with pytest.raises(ValueError, match="masked_attention"):
            F.masked_attention(b, b, b, m, **bad)
    with pytest.raises(ValueError, match="masked_attention"):
        F.masked_attention(b, b[:, :3], b[:, :3], m)
