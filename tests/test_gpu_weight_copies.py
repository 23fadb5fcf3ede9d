"""Low-precision weight copies kept on a weight, on the GPU: graph captures, updates, streams."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F

pytestmark = pytest.mark.gpu


def fp4(x, w):
    return F.mxfp4_linear(x, w)


def behind_norm(x, w):
    return F.add_norm_linear(x, None, torch.ones(x.shape[1], dtype=torch.bfloat16, device="cuda"), w)[0]


def operands(T, N=512, K=256):
    torch.manual_seed(T)
    return torch.randn(T, K, device="cuda").bfloat16(), torch.randn(N, K, device="cuda").bfloat16()


def poison():
    """Memory that the allocator hands out next holds NaN scales."""
    torch.cuda.synchronize()
    junk = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 22) for _ in range(8)]
    torch.cuda.synchronize()
    return junk


def capture(layer, x, w):
    """The layer captured; run once on other operands before, as a capture wants its kernels loaded."""
    layer(x, w.detach().clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x, w)
    return g, y


@pytest.mark.parametrize("layer", [fp4, behind_norm])
@pytest.mark.parametrize("frozen", [True, False])
def test_copies_recorded_by_a_capture_are_not_kept(layer, frozen):
    """An eager call and a second capture between a capture and its first replay make their own."""
    x, w = operands(128)
    want = layer(x, w.clone())
    w.requires_grad_(not frozen)
    with torch.no_grad():
        g, y = capture(layer, x, w)
        y.fill_(float("nan"))
        assert torch.equal(layer(x, w), want)
        g2, y2 = capture(layer, x, w)
        g2.replay()
        assert torch.equal(y2, want)
        g.replay()
        assert torch.equal(y, want)
    _lib.check_status("capture")


@pytest.mark.parametrize("layer", [fp4, behind_norm])
def test_a_graph_does_not_read_copies_made_outside_it(layer):
    """They may be gone when it is replayed, and a replay follows the weight as it does with any tensor."""
    x, w = operands(128)
    want = layer(x, w)
    torch.cuda.synchronize()
    g, y = capture(layer, x, w)
    w.mul_(-1)
    assert torch.equal(layer(x, w), -want)              # (the copies that the first call left are replaced)
    junk = poison()
    g.replay()
    assert torch.equal(y, -want)
    del junk


def test_copies_of_the_linear_behind_a_norm_made_on_one_stream_and_used_on_others():
    torch.manual_seed(0)
    x, w = torch.randn(128, 4096, device="cuda").bfloat16(), torch.randn(16384, 4096, device="cuda").bfloat16()
    want = behind_norm(x, w.clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        w = w.clone()
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(behind_norm(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
