"""Low-precision weight copies kept on a weight: what they follow (CPU)."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import linear as L


def fp4(x, w):
    return F.mxfp4_linear(x, w)


def behind_norm(x, w):
    return F.add_norm_linear(x, None, torch.ones(x.shape[1]), w)[0]


def operands():
    torch.manual_seed(0)
    return torch.randn(128, 128), torch.nn.Parameter(torch.randn(256, 128))


@pytest.mark.parametrize("layer", [fp4, behind_norm])
def test_copies_follow_other_storage(layer):
    """New storage under the same tensor (``.data``, ``Module.to`` and its relatives), another layout of the same storage."""
    x, w = operands()
    y = layer(x, w).detach()
    w.data = -w.data
    assert torch.equal(layer(x, w), -y)
    m = torch.nn.Module()
    m.w = w
    m._apply(lambda t: -t)
    assert torch.equal(layer(x, m.w), y)
    square = torch.randn(128, 128)
    v = square.clone()
    layer(x, v)
    v.data = v.data.t()                          # same pointer and shape, other strides
    assert torch.equal(layer(x, v), layer(x, v.detach().clone()))


@pytest.mark.parametrize("layer", [fp4, behind_norm])
def test_an_address_that_comes_back_is_another_storage(layer):
    x, w = operands()
    y = layer(x, w).detach()
    held = w.detach().numpy().copy()
    w.data = torch.from_numpy(held)
    layer(x, w)
    held *= -1
    w.data = torch.from_numpy(held)
    assert torch.equal(layer(x, w), -y)


@pytest.mark.parametrize("layer", [fp4, behind_norm])
def test_copies_follow_updates_in_place(layer):
    x, w = operands()
    y = layer(x, w).detach()
    for t in (w, torch.nn.Parameter(w.detach().clone(), requires_grad=False), w.detach().clone()):
        assert torch.equal(layer(x, t), y)
        with torch.no_grad():
            t.mul_(-1)
        assert torch.equal(layer(x, t), -y)
    w = torch.nn.Parameter(w.detach().clone())
    opt = torch.optim.SGD([w], lr=2.0)
    layer(x, w)
    w.grad = w.detach().clone()                  # a step of 2 w: the weight changes its sign
    opt.step()
    assert torch.equal(layer(x, w), y)           # (w was -w0)
    with torch.inference_mode():
        v = w.detach().clone()
        assert torch.equal(layer(x, v), y)
        v.mul_(-1)
        assert torch.equal(layer(x, v), -y)


def test_gradients_read_the_copies_of_the_updated_weight():
    x, w = operands()
    x.requires_grad_()
    dy = torch.randn(128, 256)
    (dx,) = torch.autograd.grad(behind_norm(x, w), x, dy)
    with torch.no_grad():
        w.mul_(-1)
    assert torch.equal(torch.autograd.grad(behind_norm(x, w), x, dy)[0], -dx)


def test_sharded_parameter_engine_knows_both_kinds_of_copies():
    """A block whose matrices have their copies, 8-bit or 4-bit, is not gathered again; copies of an older weight do not count."""
    from types import SimpleNamespace
    from mlperf_training_b200.parallel.zero3 import Zero3Engine
    x, w8 = operands()
    w4 = torch.nn.Parameter(torch.randn(256, 128))
    block = SimpleNamespace(params=[("w_qkv", w8), ("w_proj", w4)])
    cached = lambda need_col: Zero3Engine._cached(SimpleNamespace(skip_cached=True), block, need_col)
    assert not cached(False)
    with torch.no_grad():
        behind_norm(x, w8)
        fp4(x, w4)
    assert cached(False) and not cached(True)
    x.requires_grad_()
    behind_norm(x, w8)
    fp4(x, w4)
    assert cached(True)
    with torch.no_grad():
        w4.mul_(2)
    assert not cached(False)
    fp4(x, w4)
    assert cached(True)
    L.bump_weight_epoch()
    assert not cached(False)
