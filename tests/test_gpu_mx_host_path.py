"""The micro-scaled and gated operators with the native host module and without it (arguments through ctypes and Python): the same results."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX
from mlperf_training_b200.ops.norm_mx import rms_norm_quantize

pytestmark = pytest.mark.gpu


def everything(T, D, N):
    g = torch.Generator(device="cuda").manual_seed(T + D + N)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    x, r, w, wt, wd = n(T, D), n(T, D), n(D), n(2 * N, D), n(D, N)
    u = torch.randint(0, 256, (T, D), generator=g, device="cuda", dtype=torch.uint8)
    out = []
    for kw in (dict(row_tile=128), dict(col_tile=M4.b_tile(D)), dict(row_tile=128, col_tile=M4.b_tile(D), noise=u, hadamard=True)):
        out += [M4.dequantize(op, dt) for op in M4.quantize(x, **kw) if op is not None for dt in (torch.float32, torch.bfloat16)]
    for res in (None, r):
        row, col, h, rstd = rms_norm_quantize(x, w, residual=res, row_tile=MX.A_TILE, col_tile=MX.b_tile(D))
        out += [M4.dequantize(row), M4.dequantize(col), h, rstd]
        assert (h is x) == (res is None)
    out.append(F.mxfp4_linear(x, wt, bias=n(2 * N), residual=n(T, 2 * N)))
    out.append(F.mxfp4_linear(x, wt))
    a, gu = K.gated_fwd(x, wt, "gelu")
    out += [a, gu, K.gated_fwd(x, wt, want_gu=False)[0], *K.gated_bwd(r, wd, gu, "gelu"), F.gated_mlp(x, wt, wd, residual=r)]
    return out


@pytest.mark.parametrize("T,D,N", [(1, 64, 8), (33, 96, 40), (200, 512, 264)])
def test_same_results_without_the_host_module(T, D, N, monkeypatch):
    if _lib.host is None:
        pytest.skip("the host module is not built")
    with_host = everything(T, D, N)
    monkeypatch.setattr(_lib, "host", None)
    without = everything(T, D, N)
    assert len(with_host) == len(without) and all(torch.equal(a, b) for a, b in zip(with_host, without))


def test_what_the_host_module_leaves_to_the_general_path():
    """Inputs that need a copy, and wrong ones, come out as without the module."""
    x = torch.randn(40, 100, device="cuda").bfloat16()[:, 2:98]
    w = torch.randn(64, 96, device="cuda").bfloat16()
    assert torch.equal(F.mxfp4_linear(x, w), F.mxfp4_linear(x.contiguous(), w))
    a = rms_norm_quantize(x, torch.ones(96, device="cuda"), row_tile=128)[0]
    b = rms_norm_quantize(x.contiguous(), torch.ones(96, device="cuda").bfloat16(), row_tile=128)[0]
    assert torch.equal(a.q, b.q)
    for bad in (lambda: M4.quantize(x, row_tile=0, col_tile=128), lambda: M4.quantize(x[:, :90], row_tile=128),
                lambda: rms_norm_quantize(x, w, row_tile=128), lambda: K.gated_fwd(x, w[:63]), lambda: K.gated_fwd(x, w, "relu"),
                lambda: F.mxfp4_linear(x, w, bias=torch.zeros(63, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
