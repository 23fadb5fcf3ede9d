"""MXFP4 operands on the CPU: the eager definitions against one written element by element in 64 bits, the linear layer's gradients
against its formula and against differences, refusals."""
import math

import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import linear as L
from mlperf_training_b200.ops import mxfp4 as M4

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def block_by_hand(block, noise=None):
    """32 Python floats -> their MXFP4 values."""
    amax = max(abs(v) for v in block)
    if any(not math.isfinite(v) for v in block):
        return [math.nan] * 32
    if amax == 0:
        return [0.0] * 32
    e = -126
    while amax > 6.0 * 2.0 ** e:
        e += 1
    out = []
    for i, v in enumerate(block):
        a = abs(v) / 2.0 ** e
        k = max(j for j in range(8) if GRID[j] <= a)
        if k < 7:
            part = (a - GRID[k]) / (GRID[k + 1] - GRID[k])
            if noise is None:
                k += part > 0.5 or (part == 0.5 and k % 2 == 1)
            else:
                k += part + (noise[i] + 0.5) / 256 >= 1
        out.append(math.copysign(GRID[k] * 2.0 ** e, v))
    return out


def edge_matrix():
    torch.manual_seed(0)
    x = torch.randn(24, 64) * torch.exp2(torch.randint(-20, 20, (24, 1)).float())
    x[0, :32] = 0
    x[1, 3] = float("inf")
    x[2, 40] = float("nan")
    x[3, :32] = torch.linspace(-6, 6, 32)
    x[4, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)       # ties
    x[5, :32] = 1.5 * 2.0 ** 10                                                      # amax on the boundary of a scale, and above it
    x[6, :32] = 1.5 * 2.0 ** 10 * (1 + 2 ** -7)
    x[7, :32] = 2.0 ** -133                                                          # a bf16 denormal
    x[8, :32] = 3.3e38
    return x.bfloat16()


@pytest.mark.parametrize("stochastic", [False, True])
def test_quantize_by_hand(stochastic):
    x = edge_matrix()
    u = torch.randint(0, 256, x.shape, dtype=torch.uint8) if stochastic else None
    row, col = M4.quantize(x, row_tile=128, col_tile=128, noise=u)
    got = M4.dequantize(row)
    for r in range(x.shape[0]):
        for b in range(0, 64, 32):
            want = block_by_hand(x[r, b:b + 32].tolist(), None if u is None else u[r, b:b + 32].tolist())
            assert torch.equal(got[r, b:b + 32].nan_to_num(9e9), torch.tensor(want).nan_to_num(9e9)), (r, b)
    assert (col.rows, col.k) == (64, 32)
    got = M4.dequantize(col)
    for c in range(64):
        v = x[:, c].tolist() + [0.0] * 8
        want = block_by_hand(v, None if u is None else u[:, c].tolist() + [128] * 8)
        assert torch.equal(got[c].nan_to_num(9e9), torch.tensor(want).nan_to_num(9e9)), c


def test_pack_holds_the_even_element_low():
    x = torch.zeros(1, 32)
    x[0, 0], x[0, 1], x[0, 31] = 6.0, -0.5, 1.0
    op = M4.quantize(x, row_tile=128)[0]
    assert int(op.q[0, 0]) == 0x97 and int(op.q[0, 15]) == 0x20 and int(op.sf[0, 0]) == 127


def test_stochastic_rounding_averages_to_the_input():
    """The mean over all 256 bytes is the input to within half a byte's step of a quantum (2 s): s / 256."""
    x = torch.linspace(-6, 6, 32)[None].repeat(256, 1)
    u = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 32)
    mean = M4.dequantize(M4.quantize(x, row_tile=128, noise=u)[0]).double().mean(0)
    assert float((mean - x[0].double()).abs().max()) <= 2 / 512 + 1e-6


def test_hadamard_leaves_the_product():
    torch.manual_seed(1)
    a, b = torch.randn(48, 7).double(), torch.randn(48, 5).double()
    assert torch.allclose(M4.hadamard16(a).t() @ M4.hadamard16(b), a.t() @ b, atol=1e-12)


@pytest.mark.parametrize("T", [1, 40, 64])
def test_linear_is_its_formula(T):
    torch.manual_seed(T)
    x = torch.randn(T, 64, requires_grad=True)
    w = torch.randn(96, 64, requires_grad=True)
    b, r = torch.randn(96, requires_grad=True), torch.randn(T, 96, requires_grad=True)
    u = torch.randint(0, 256, (T, 96), dtype=torch.uint8)
    dy = torch.randn(T, 96)
    y = F.mxfp4_linear(x, w, b, r, u)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], dy)
    q = lambda v, **kw: M4.dequantize(M4.quantize(v, row_tile=128, **kw)[0])
    qt = lambda v, **kw: M4.dequantize(M4.quantize(v, col_tile=128, **kw)[1])
    x, w = x.detach(), w.detach()
    assert torch.allclose(y, q(x) @ q(w).t() + b + r, atol=1e-5)
    assert torch.allclose(dx, q(dy, noise=u) @ qt(w).t(), atol=1e-5)
    assert torch.allclose(dw, qt(dy, noise=u, hadamard=True) @ qt(x, hadamard=True).t(), atol=1e-4)
    assert torch.allclose(db, dy.sum(0), atol=1e-5) and torch.equal(dr, dy)


def test_linear_gradients_point_where_differences_do():
    """On operands that 4 bits hold exactly the layer is a linear map: differences of it are its gradient's formula without rounding; the
    rounded gradient lies within the format's resolution of it (a quarter of a value, so its cosine is above 0.95)."""
    torch.manual_seed(3)
    pick = lambda *s: torch.tensor(GRID)[torch.randint(0, 8, s)] * (1 - 2 * torch.randint(0, 2, s))
    x, w, dy = pick(32, 32), pick(64, 32), torch.randn(32, 64)
    f = lambda x, w: float((F.mxfp4_linear(x, w).double() * dy.double()).sum())
    with torch.no_grad():
        x[:, 0], w[:, 0] = 6.0, 6.0                     # every block keeps the scale 1
        e = torch.zeros_like(x)
        e[3, 5] = (2.0 if x[3, 5] <= 2 else -2.0) if x[3, 5] in (0, 2, 4) else -float(x[3, 5])
        e[3, 5] = e[3, 5] or 1.0
        slope = (f(x + e, w) - f(x, w)) / float(e[3, 5])
        assert abs(slope - float((dy @ w)[3, 5])) < 1e-3
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(F.mxfp4_linear(xg, wg), [xg, wg], dy)
    cos = lambda a, b: float(torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), 0))
    assert cos(dx, dy @ w) > 0.95 and cos(dw, dy.t() @ x) > 0.95


def test_main_grad_and_frozen_weight():
    torch.manual_seed(4)
    x, w = torch.randn(32, 64, requires_grad=True), torch.nn.Parameter(torch.randn(32, 64))
    u = torch.randint(0, 256, (32, 32), dtype=torch.uint8)
    (want,) = torch.autograd.grad(F.mxfp4_linear(x, w, noise=u).sum(), w)
    w.main_grad = torch.ones(32, 64)
    F.mxfp4_linear(x, w, noise=u).sum().backward()
    assert w.grad is None and torch.allclose(w.main_grad, 1 + want, atol=1e-5)
    w2 = torch.randn(32, 64)
    y0 = F.mxfp4_linear(x, w2)
    w2.mul_(-1)                                          # an update in place: the kept copies are not used again
    assert torch.equal(F.mxfp4_linear(x, w2), -y0)


def test_weight_copies_follow_the_optimizer_epoch():
    w = torch.nn.Parameter(torch.randn(32, 32))
    x = torch.randn(4, 32)
    y0 = F.mxfp4_linear(x, w)
    w.data.mul_(-1)                                      # past autograd's version counter
    L.bump_weight_epoch()
    assert torch.equal(F.mxfp4_linear(x, w), -y0)


def test_deoscillation_tracks_the_4_bit_weights():
    """In the fp4 recipe the weights with 4-bit copies are tracked, and nothing else; one that flips between two codes is put on the grid."""
    from mlperf_training_b200.ops.recipe import DeoscConfig, Deoscillator
    from mlperf_training_b200.parallel.engine import OptimConfig, ZeroEngine
    torch.manual_seed(0)
    w4, w8 = torch.nn.Parameter(torch.randn(32, 64)), torch.nn.Parameter(torch.randn(32, 64))
    engine = ZeroEngine(torch.nn.ParameterList([w4, w8]), OptimConfig())
    d = Deoscillator(engine, DeoscConfig(enabled=True, start_step=0, period=8, ratio=2.0))
    assert "on" in d.cfg.status("fp4") and "idle" in d.cfg.status("mxfp8")
    with torch.no_grad():
        w4[0, :32], w8[0, :32] = 6.0, 6.0
        F.mxfp4_linear(torch.randn(1, 64), w4)
        for step in range(8):
            for b in engine.buckets:
                for (name, p), o in zip(b.params, b.offsets):
                    at = 1 if p is w4 or p is w8 else None
                    if at is not None and b.master is not None:
                        b.master[o - b.lo + at] = 2.5 + (0.1 if step % 2 else -0.1)
                    p[0, 1] = 2.5 + (0.1 if step % 2 else -0.1)
            n = d.after_step(step, "fp4")
        assert n == 1 and float(w4[0, 1]) in (2.0, 3.0) and float(w8[0, 1]) not in (2.0, 3.0)


def test_gemm_edges():
    a = M4.quantize(torch.randn(3, 32), row_tile=128)[0]
    b = M4.quantize(torch.randn(5, 32), row_tile=128)[0]
    ref = M4.dequantize(a) @ M4.dequantize(b).t()
    out = torch.ones(3, 5)
    M4.gemm(a, b, out=out, accumulate=True, alpha=2.0)
    assert torch.allclose(out, 1 + 2 * ref, atol=1e-5)
    empty = M4.quantize(torch.randn(0, 32), row_tile=128, col_tile=128)
    assert M4.gemm(empty[0], b).shape == (0, 5)
    assert torch.equal(M4.gemm(empty[1], empty[1], bias=torch.ones(32), out_dtype=torch.float32), torch.ones(32, 32))


def test_refusals():
    x, op = torch.randn(4, 32), M4.quantize(torch.randn(4, 32), row_tile=128)[0]
    wide = M4.quantize(torch.randn(4, 64), row_tile=128)[0]
    for bad in (lambda: M4.quantize(torch.randn(4, 33), row_tile=128), lambda: M4.quantize(torch.randn(32), row_tile=128),
                lambda: M4.quantize(x, row_tile=100), lambda: M4.quantize(x, row_tile=128, noise=torch.zeros(4, 31, dtype=torch.uint8)),
                lambda: M4.quantize(x, row_tile=128, noise=torch.zeros(4, 32)), lambda: M4.gemm(op, wide),
                lambda: M4.gemm(op, op, accumulate=True), lambda: M4.gemm(op, op, out=torch.zeros(4, 5)),
                lambda: M4.gemm(op, op, bias=torch.zeros(5)), lambda: M4.gemm(op, op, residual=torch.zeros(4, 5)),
                lambda: F.mxfp4_linear(torch.randn(4, 33), torch.randn(32, 33)), lambda: F.mxfp4_linear(x, torch.randn(32, 64)),
                lambda: F.mxfp4_linear(x.clone().requires_grad_(), torch.randn(5, 32)),
                lambda: F.mxfp4_linear(x, torch.nn.Parameter(torch.randn(5, 32))),
                lambda: F.mxfp4_linear(x, torch.randn(32, 32), noise=torch.zeros(4, 32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        M4.gemm(op, torch.randn(4, 32))
    with pytest.raises(TypeError):
        M4.dequantize(op, torch.float16)
    assert F.mxfp4_linear(x, torch.randn(5, 32)).shape == (4, 5)         # any width without a gradient
