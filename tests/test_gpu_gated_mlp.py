"""Gated feed-forward block on the GPU: both fused kernels against 64 bits and against the separate kernels, the whole block's gradients."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
ACT = {"silu": torch.nn.functional.silu, "gelu": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}
SIZES = [(1, 8, 8), (1, 256, 136), (7, 4096, 1000), (128, 264, 128), (257, 64, 120), (300, 520, 392), (1000, 512, 1032), (2048, 1024, 2880)]


def make(T, D, Fh, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + D + Fh)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return n(T, D).bfloat16(), (n(2 * Fh, D) * D ** -0.5 * 2).bfloat16(), (n(D, Fh) * Fh ** -0.5).bfloat16(), n(T, D).bfloat16()


@pytest.mark.parametrize("T,D,Fh", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_kernels_against_64_bits(T, D, Fh, act):
    """Each element within its one rounding to bf16 (2^-9), and 1e-5 of the largest for the sums and the activation."""
    x, w, wd, dy = make(T, D, Fh)
    a, gu = K.gated_fwd(x, w, act)
    a2, none = K.gated_fwd(x, w, act, want_gu=False)
    assert none is None and torch.equal(a, a2)
    g, u = (x.double() @ w.double().t()).chunk(2, 1)
    want = torch.cat([g, u], 1)
    assert bool(((gu.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5 * want.abs().max()).all())
    want = ACT[act](g) * u
    assert bool(((a.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5 * want.abs().max()).all())
    gr, ur = gu.double().chunk(2, 1)
    gr.requires_grad_()
    v = ACT[act](gr)
    dgu, a3 = K.gated_bwd(dy, wd, gu, act)
    want = (v * ur).detach()
    assert bool(((a3.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5 * want.abs().max()).all())
    assert torch.equal(K.gated_bwd(dy, wd, gu, act, want_a=False)[0], dgu)
    da = dy.double() @ wd.double()
    (dg,) = torch.autograd.grad(v, gr, da * ur)
    want = torch.cat([dg, da * v.detach()], 1)
    assert bool(((dgu.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5 * want.abs().max()).all())
    _lib.check_status("gated")


@pytest.mark.parametrize("T,D,Fh", SIZES)
def test_block_and_gradients(T, D, Fh):
    x, w, wd, r = make(T, D, Fh, 1)
    t = [v.clone().requires_grad_() for v in (x, w, wd, r)]
    y = F.gated_mlp(*t)
    dy = torch.randn(T, D, device="cuda").bfloat16()
    got = torch.autograd.grad(y, t, dy)
    d = [v.double().requires_grad_() for v in (x, w, wd, r)]
    g, u = (d[0] @ d[1].t()).chunk(2, 1)
    yd = (torch.nn.functional.silu(g) * u) @ d[2].t() + d[3]
    with torch.no_grad():
        assert torch.equal(F.gated_mlp(*t), y)
    # a few roundings of 2^-9 each along every path
    assert float((y.double() - yd).norm() / yd.norm()) < 2 ** -7
    for a, b in zip(got, torch.autograd.grad(yd, d, dy.double())):
        assert float((a.double() - b).norm() / b.norm()) < 2 ** -6


def test_same_as_the_separate_kernels():
    """Against the GEMM and the element-wise kernels: the projections but for the last bit of a sum, the rest to a rounding or two more."""
    x, w, wd, dy = make(512, 512, 1024)
    gu = K.gemm(x, w)
    a, gu2 = K.gated_fwd(x, w)
    assert float((gu != gu2).float().mean()) < 1e-2
    ref = K.swiglu_fwd(gu2).float()
    assert float((ref - a.float()).norm() / ref.norm()) < 2 ** -7
    da = K.gemm(dy, wd, b_mn_major=True)
    dgu, _ = K.gated_bwd(dy, wd, gu2)
    ref = K.swiglu_bwd(da, gu2)
    assert float((dgu.float() - ref.float()).norm() / ref.float().norm()) < 2 ** -7


def test_extreme_gates_and_non_finite_rows():
    """Gates far past where the exponentials end give 0 or the up projection, with finite gradients; a row with a NaN or an infinity stays apart."""
    for act in ("silu", "gelu"):
        x = torch.zeros(300, 64, device="cuda").bfloat16()
        x[:, 0] = torch.linspace(-3e4, 3e4, 300, device="cuda").bfloat16()
        w = torch.zeros(2 * 128, 64, device="cuda").bfloat16()
        w[:128, 0], w[128:, 1] = 1.0, 1.0
        x[:, 1] = 1.0
        a, gu = K.gated_fwd(x, w, act)
        want = torch.where(x[:, :1].double() > 0, x[:, :1].double(), torch.zeros((), device="cuda", dtype=torch.float64)).expand(300, 128)
        assert bool(((a.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-3).all())
        dgu, _ = K.gated_bwd(torch.ones(300, 64, device="cuda").bfloat16(), torch.ones(64, 128, device="cuda").bfloat16(), gu, act)
        assert bool(dgu.isfinite().all())
        x[5, 2], x[290, 3] = float("nan"), float("inf")
        w[:, 2], w[:, 3] = 0.5, 0.5
        a, _ = K.gated_fwd(x, w, act)
        clean = torch.ones(300, dtype=torch.bool, device="cuda")
        clean[[5, 290]] = False
        assert bool(a[clean].isfinite().all()) and bool(a[5].isnan().all()) and not bool(a[290].isfinite().any())


def test_strides_streams_and_no_tokens():
    x, w, wd, dy = make(100, 64, 72)
    wide = torch.zeros(100, 80, device="cuda").bfloat16()
    wide[:, 8:72] = x
    odd = torch.zeros(100, 67, device="cuda").bfloat16()
    odd[:, 3:] = x
    want = F.gated_mlp(x, w, wd)
    assert torch.equal(F.gated_mlp(wide[:, 8:72], w, wd), want) and torch.equal(F.gated_mlp(odd[:, 3:], w, wd), want)
    assert torch.equal(F.gated_mlp(x, w.t().contiguous().t(), wd.t().contiguous().t()), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.gated_mlp(x, w, wd)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    e, p = x[:0].clone().requires_grad_(), torch.nn.Parameter(w.clone())
    F.gated_mlp(e, p, wd).sum().backward()
    assert e.grad.shape == (0, 64) and float(p.grad.abs().max()) == 0.0


def test_refusals():
    x, w, wd, _ = make(4, 64, 72)
    with pytest.raises(TypeError):
        F.gated_mlp(x.float(), w.float(), wd.float())
    with pytest.raises(ValueError):
        F.gated_mlp(x, w[:2 * 68], wd[:, :68])
    with pytest.raises(ValueError):
        F.gated_mlp(x[:, :60], w[:, :60], wd)
    with pytest.raises(ValueError):
        F.gated_mlp(x.cpu(), w, wd)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        _lib.call("b200_gemm_gated", x.data_ptr(), w.data_ptr(), x.data_ptr(), None, 4, 12, 64, 64, 64, 16, 0, 0, _lib.stream_ptr())


@pytest.mark.parametrize("T", [1, 7, 8, 16, 17, 33, 64])
@pytest.mark.parametrize("N,Fh", [(8, 8), (136, 64), (128, 72), (264, 1000), (1000, 1032), (512, 2056), (4096, 14336), (19008, 512)])
def test_down_projection_of_few_rows(T, N, Fh):
    """Against 64 bits: the one rounding to bf16 (2^-9, doubled for a sum near a boundary), and 2^-23 of the running sum, taken as twice the
    largest result, for each of the Fh / 16 steps of the accumulation.  The same result every time; strided and broadcast residuals."""
    g = torch.Generator(device="cuda").manual_seed(T + N + Fh)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    a, w, r = n(T, Fh).bfloat16(), (n(N, Fh) * Fh ** -0.5).bfloat16(), n(T, N).bfloat16()
    wide = torch.zeros(T, N + 16, device="cuda").bfloat16()
    wide[:, 8:N + 8] = r
    for res in (None, r, wide[:, 8:N + 8], r[:1].expand(T, N)):
        y = K.gated_down(a, w, res)
        want = a.double() @ w.double().t() + (0 if res is None else res.double())
        assert bool(((y.double() - want).abs() <= want.abs() * 2 ** -8 + max(1, Fh / 16) * 2 ** -22 * want.abs().max()).all())
        assert torch.equal(K.gated_down(a, w, res), y)
    _lib.check_status("gated_down")


def test_down_projection_keeps_rows_apart_and_leaves_neighbours_alone():
    """A row with a NaN or an infinity stays apart; a weight row too; operands inside larger buffers filled with NaN."""
    T, N, Fh = 9, 200, 1096
    big_a = torch.full((T + 8, Fh + 64), float("nan"), device="cuda").bfloat16()
    big_w = torch.full((N + 128, Fh + 64), float("nan"), device="cuda").bfloat16()
    big_a[:T, :Fh] = torch.randn(T, Fh, device="cuda").bfloat16()
    big_w[:N, :Fh] = torch.randn(N, Fh, device="cuda").bfloat16()
    a, w = big_a[:T, :Fh], big_w[:N, :Fh]
    y = K.gated_down(a, w)
    assert bool(y.isfinite().all()) and torch.equal(y, K.gated_down(a.contiguous(), w.contiguous()))
    a[3, 1095], w[150, 0] = float("nan"), float("inf")
    z = K.gated_down(a, w)
    keep = torch.ones(T, N, dtype=torch.bool, device="cuda")
    keep[3], keep[:, 150] = False, False
    assert torch.equal(z[keep], y[keep]) and bool(z[3].isnan().all()) and not bool(z[:, 150].isfinite().any())


def test_down_projection_refusals_and_more_rows():
    a, w = torch.randn(4, 64, device="cuda").bfloat16(), torch.randn(72, 64, device="cuda").bfloat16()
    for bad in (lambda: K.gated_down(a, w[:, :56]), lambda: K.gated_down(a, w[:71]), lambda: K.gated_down(a, w.cpu()),
                lambda: K.gated_down(a, w, torch.zeros(4, 64, device="cuda").bfloat16())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        K.gated_down(a, w.float())
    with pytest.raises(RuntimeError, match="1 to 64 rows"):
        _lib.call("b200_gated_down", a.data_ptr(), w.data_ptr(), None, a.data_ptr(), 65, 72, 64, 64, 64, 0, 72, _lib.stream_ptr())
    many = torch.randn(65, 64, device="cuda").bfloat16()
    assert torch.equal(K.gated_down(many, w), K.gemm(many, w))
