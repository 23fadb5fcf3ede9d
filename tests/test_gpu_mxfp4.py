"""MXFP4 kernels on the GPU: quantiser and dequantiser against the eager definition (bit for bit), the product against 64 bits, the linear
layer, other streams and strides, refusals at the launcher."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import linear as L
from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX

pytestmark = pytest.mark.gpu


def poison(n=1 << 24):
    """Freed memory full of 255: a scale byte that nothing wrote would be a NaN."""
    for k in (n, n // 16, 4096):
        del_me = torch.full((k,), 255, dtype=torch.uint8, device="cuda")
        del del_me


def same(a, b):
    return a.shape == b.shape and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


@pytest.mark.parametrize("R,C", [(1, 32), (15, 64), (31, 96), (33, 160), (128, 128), (257, 416), (515, 2880)])
@pytest.mark.parametrize("stochastic", [False, True])
@pytest.mark.parametrize("hadamard", [False, True])
def test_quantize_is_the_definition(R, C, stochastic, hadamard):
    torch.manual_seed(R + C)
    x = (torch.randn(R, C) * torch.exp2(torch.randint(-30, 30, (R, 1)).float())).bfloat16()
    x[0, :32] = 0
    if R > 14:
        x[3, 1], x[4, 2], x[5, 3] = float("inf"), float("-inf"), float("nan")
        x[6, :32], x[7, :32], x[8, :32] = 1.5 * 2.0 ** 100, 2.0 ** -133, 3.3e38
        x[9, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)
    if hadamard:
        x[:] = (x.float().nan_to_num(1.0, 1.0, 1.0).clamp(-8, 8) * 64).round() / 64      # sums of sixteen that fp32 holds exactly, in any order
    u = torch.randint(0, 256, (R, C), dtype=torch.uint8) if stochastic else None
    ug = None if u is None else u.cuda()
    want = M4.quantize(x, row_tile=M4.A_TILE, col_tile=M4.b_tile(C), noise=u, hadamard=hadamard)
    poison()
    got = M4.quantize(x.cuda(), row_tile=M4.A_TILE, col_tile=M4.b_tile(C), noise=ug, hadamard=hadamard)
    for a, b, what in zip(want, got, ("row", "column")):
        assert torch.equal(a.sf, M4.sf_plain(b).cpu()), f"{what} scales"
        assert same(M4.dequantize(a), M4.dequantize(b).cpu()), f"{what} values"
        assert same(M4.dequantize(a, torch.bfloat16), M4.dequantize(b, torch.bfloat16).cpu())
        # what fills the last scale word of a row is written, as zero
        pad = (b.k + 127) // 128 * 128
        full = b.sf[MX.sf_index(b.rows, pad, b.tile_rows, "cuda")]
        assert int(full[:, b.k // 32:].sum()) == 0
    only = M4.quantize(x.cuda(), col_tile=M4.b_tile(C), noise=ug, hadamard=hadamard)
    assert only[0] is None and torch.equal(only[1].q, got[1].q)
    _lib.check_status("quantize")


def test_quantize_strided_and_misaligned_inputs():
    torch.manual_seed(0)
    base = torch.randn(70, 200, device="cuda").bfloat16()
    noise = torch.randint(0, 256, (70, 201), dtype=torch.uint8, device="cuda")
    for x, u in ((base[:, 8:104], noise[:, 5:101]), (base[:, 3:99], noise[:, :96]), (base[::2, :96], noise[::2, 1:97]),
                 (base.t()[8:104, :64], noise.t()[7:103, :64]), (base[:1].expand(70, 200)[:, :192], noise[:, :192])):
        a = M4.quantize(x, row_tile=128, col_tile=128, noise=u, hadamard=True)
        b = M4.quantize(x.clone().contiguous(), row_tile=128, col_tile=128, noise=u.clone().contiguous(), hadamard=True)
        assert all(torch.equal(p.q, q.q) and torch.equal(M4.sf_plain(p), M4.sf_plain(q)) for p, q in zip(a, b))


def test_dequantize_of_8_bit_operands():
    x = torch.randn(128, 96, device="cuda").bfloat16()
    for op in MX.quantize(x, row_tile=MX.A_TILE, col_tile=MX.b_tile(96)):
        assert torch.equal(M4.dequantize(op), MX.dequantize(op))


def operands(M, N, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn(M, K, generator=g, device="cuda") * torch.exp2(torch.randint(-4, 5, (M, 1), generator=g, device="cuda").float())
    b = torch.randn(N, K, generator=g, device="cuda")
    poison()
    a = M4.quantize(a.bfloat16(), row_tile=M4.A_TILE)[0]
    b = M4.quantize(b.bfloat16(), row_tile=M4.b_tile(N))[0]
    return a, b, M4.dequantize(a).double() @ M4.dequantize(b).double().t()


@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (1, 1, 32), (5, 7, 64), (128, 128, 96), (129, 129, 128), (255, 191, 160), (256, 192, 256), (257, 193, 288),
                                   (1, 4096, 4096), (64, 513, 14336), (300, 1000, 2880), (2003, 640, 992), (1024, 1024, 4096)])
def test_product(M, N, K):
    """fp32 output against 64 bits: the products of 64 codes are summed exactly, the sums and their accumulation have 24 bits - at most
    K / 64 roundings of a sum, none above the largest partial sum.  1e-5 of the row's root-sum-square of products covers K = 14336."""
    a, b, ref = operands(M, N, K, M + N + K)
    bound = 1e-5 * (M4.dequantize(a).double().square() @ M4.dequantize(b).double().square().t()).sqrt() + 1e-30
    d = M4.gemm(a, b, out_dtype=torch.float32)
    _lib.check_status("gemm_mxfp4")
    assert d.shape == (M, N) and bool(((d.double() - ref).abs() <= bound).all())
    h = M4.gemm(a, b)
    assert h.dtype == torch.bfloat16 and bool(((h.double() - ref).abs() <= bound + ref.abs() * 2 ** -8).all())


@pytest.mark.parametrize("M,N,K", [(7, 24, 64), (300, 203, 288), (512, 4096, 8192)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_epilogues(M, N, K, dtype):
    """alpha, bias, residual and accumulation; outputs that are views of wider rows, misaligned rows and columns among them."""
    a, b, ref = operands(M, N, K, 1)
    ref = ref / K ** 0.5
    bias, res = torch.randn(N, device="cuda").bfloat16(), torch.randn(M, N + 8, device="cuda").bfloat16()[:, :N]
    want = ref + bias.double() + res.double()
    tol = lambda w: 2 ** (-7 if dtype == torch.bfloat16 else -20) * (w.abs() + float(ref.abs().max())) + 1e-6
    d = M4.gemm(a, b, out_dtype=dtype, bias=bias, residual=res, alpha=K ** -0.5)
    assert bool(((d.double() - want).abs() <= tol(want)).all())
    for cols, off in ((N + 16, 8), (N + 5, 0), (N + 3, 1)):
        wide = torch.full((M, cols), 3.0, dtype=dtype, device="cuda")
        out = wide[:, off:off + N]
        assert M4.gemm(a, b, out=out, accumulate=True, alpha=K ** -0.5) is out
        assert bool(((out.double() - ref - 3).abs() <= tol(ref + 3)).all())
        M4.gemm(a, b, out=out, alpha=K ** -0.5)
        assert bool(((out.double() - ref).abs() <= tol(ref)).all())
        keep = torch.ones(cols, dtype=torch.bool, device="cuda")
        keep[off:off + N] = False
        assert bool((wide[:, keep] == 3).all())


def test_product_carries_nan_and_inf_in_their_rows_alone():
    a, b, ref = operands(300, 200, 256, 5)
    x = M4.dequantize(a)
    x[7, 40], x[280, 255] = float("nan"), float("inf")
    bad = M4.quantize(x.bfloat16(), row_tile=128)[0]
    d = M4.gemm(bad, b, out_dtype=torch.float32)
    rows = torch.zeros(300, dtype=torch.bool, device="cuda")
    rows[[7, 280]] = True
    assert bool(d[rows].isnan().all()) and bool(d[~rows].isfinite().all())


def test_empty_sizes():
    b = M4.quantize(torch.randn(40, 32, device="cuda").bfloat16(), row_tile=M4.b_tile(40))[0]
    row, col = M4.quantize(torch.zeros(0, 32, device="cuda", dtype=torch.bfloat16), row_tile=128, col_tile=128)
    assert M4.gemm(row, b).shape == (0, 40) and M4.dequantize(row).shape == (0, 32)
    out = torch.ones(32, 32, device="cuda")
    M4.gemm(col, col, out=out, accumulate=True)
    assert torch.equal(out, torch.ones_like(out))


@pytest.mark.parametrize("T,N,K", [(1, 32, 32), (77, 96, 160), (256, 512, 384), (1111, 2880, 512)])
def test_linear_matches_the_eager_layer(T, N, K):
    """Same operands bit for bit (inputs whose transforms are exact), so the products differ by fp32 sums and one rounding to bf16."""
    torch.manual_seed(T)
    grid = lambda *s: ((torch.randn(*s) * 16).round() / 16).bfloat16()
    x, w, dy, r, b = grid(T, K), grid(N, K), grid(T, N), grid(T, N), grid(N)
    u = torch.randint(0, 256, (T, N), dtype=torch.uint8)
    out = []
    for dev in ("cpu", "cuda"):
        t = [v.to(dev).requires_grad_() for v in (x, w, b, r)]
        y = F.mxfp4_linear(t[0], t[1], t[2], t[3], u.to(dev))
        out.append([y] + list(torch.autograd.grad(y, t, dy.to(dev))))
    _lib.check_status("mxfp4_linear")
    for c, g in zip(*([t.detach() for t in o] for o in out)):
        assert g.dtype == torch.bfloat16 and float((g.cpu().float() - c.float()).norm()) <= 2 ** -8 * float(c.float().norm())


def test_linear_on_another_stream_and_after_updates():
    torch.manual_seed(0)
    x, w = torch.randn(64, 256, device="cuda").bfloat16(), torch.randn(512, 256, device="cuda").bfloat16()
    want = F.mxfp4_linear(x, w.clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.mxfp4_linear(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    w.mul_(-1)
    assert torch.equal(F.mxfp4_linear(x, w), -want)
    with torch.inference_mode():
        wi = torch.randn(512, 256, device="cuda").bfloat16()
        y0 = F.mxfp4_linear(x, wi)
        wi.mul_(-1)
        assert torch.equal(F.mxfp4_linear(x, wi), -y0)


def test_weight_copies_made_on_one_stream_and_used_on_others():
    """The copies that a first call leaves on the weight are complete before another stream's call reads them."""
    torch.manual_seed(0)
    x, w = torch.randn(8, 4096, device="cuda").bfloat16(), torch.randn(16384, 4096, device="cuda").bfloat16()
    want = F.mxfp4_linear(x, w.clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        w = w.clone()
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(F.mxfp4_linear(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_linear_in_a_graph():
    """Capture and replay of the layer: the copies of a frozen weight that a call made before are read, new inputs give new outputs."""
    torch.manual_seed(0)
    x, w = torch.randn(33, 256, device="cuda").bfloat16(), torch.randn(512, 256, device="cuda").bfloat16()
    F.mxfp4_linear(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = F.mxfp4_linear(x, w)
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        g.replay()
        assert torch.equal(y, F.mxfp4_linear(x, w))


def test_drawn_noise_is_fresh_and_unbiased():
    """The backward draws its bytes itself when none are given: two backward passes differ, and their mean approaches the product with the
    unrounded gradient (256 draws: 1/16 of one draw's error)."""
    torch.manual_seed(0)
    x, w = torch.randn(32, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(64, 64, device="cuda").bfloat16()
    dy = torch.randn(32, 64, device="cuda").bfloat16()
    w_col = M4.dequantize(L.fp4_weight_operands(w)[1])
    ref = dy.float() @ w_col.t()
    draws = torch.stack([torch.autograd.grad(F.mxfp4_linear(x, w), x, dy)[0].float() for _ in range(256)])
    one = float((draws[0] - ref).norm() / ref.norm())
    assert not torch.equal(draws[0], draws[1])
    assert float((draws.mean(0) - ref).norm() / ref.norm()) < one / 8


def test_runs_are_reproducible():
    torch.manual_seed(0)
    x, w = torch.randn(500, 4096, device="cuda").bfloat16(), torch.randn(640, 4096, device="cuda").bfloat16()
    assert torch.equal(F.mxfp4_linear(x, w), F.mxfp4_linear(x, w))


def test_refusals():
    x = torch.randn(4, 32, device="cuda")
    op = M4.quantize(x.bfloat16(), row_tile=128)[0]
    with pytest.raises(TypeError):
        M4.quantize(x, row_tile=128)
    with pytest.raises(TypeError):
        M4.gemm(op, op, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        M4.gemm(op, M4.quantize(x.bfloat16(), row_tile=208)[0])
    with pytest.raises(ValueError):
        M4.gemm(op, M4.quantize(x.cpu(), row_tile=128)[0])
    with pytest.raises(ValueError):
        M4.quantize(x.bfloat16(), row_tile=128, noise=torch.zeros(4, 32, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="multiple of 32"):
        _lib.call("b200_quant_mxfp4", x.data_ptr(), 32, 4, 40, None, 0, None, None, 0, None, None, 0, _lib.stream_ptr())
    with pytest.raises(RuntimeError, match="multiple of 32"):
        _lib.call("b200_gemm_mxfp4", *[x.data_ptr()] * 5, 4, 4, 33, 16, 16, 8, 0, 0, None, None, 0, 1.0, None, 0, _lib.stream_ptr())
