"""Gated block on the GPU: what its gradients lose to rounding, and the projections kept in fp32."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
ACT = {"silu": torch.nn.functional.silu, "gelu": lambda g: torch.nn.functional.gelu(g, approximate="tanh")}
SIZES = [(1, 8, 8), (7, 256, 512), (64, 128, 136), (65, 72, 40), (300, 256, 264), (512, 512, 1024), (1000, 64, 2088)]


def make(T, D, Fh):
    torch.manual_seed(T + Fh)
    r = lambda *s: torch.randn(*s, device="cuda")
    return r(T, D).bfloat16(), (r(2 * Fh, D) * D ** -0.5).bfloat16(), (r(D, Fh) * Fh ** -0.5).bfloat16(), r(T, D).bfloat16()


@pytest.mark.parametrize("T,D,Fh", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_projections_in_fp32(T, D, Fh, act):
    """Projections to fp32 sums; the activation made again from them is the forward's bit for bit; the gradient is rounded once."""
    x, w, wd, dy = make(T, D, Fh)
    torch.full((1 << 22,), float("nan"), device="cuda")
    a, gu = K.gated_fwd(x, w, act, gu_dtype=torch.float32)
    short, gu16 = K.gated_fwd(x, w, act)
    want = x.double() @ w.double().t()
    assert gu.dtype == torch.float32 and bool(((gu.double() - want).abs() <= 1e-5 * want.abs().max()).all())
    assert torch.equal(a, short) and torch.equal(gu.bfloat16(), gu16)
    g, u = gu.double().chunk(2, 1)
    g.requires_grad_()
    v = ACT[act](g)
    da = dy.double() @ wd.double()
    (dg,) = torch.autograd.grad(v, g, da * u)
    want = torch.cat([dg, da * v.detach()], 1)
    dgu, again = K.gated_bwd(dy, wd, gu, act)
    assert torch.equal(again, a) and dgu.dtype == torch.bfloat16
    assert bool(((dgu.double() - want).abs() <= want.abs() * 2 ** -8 + 1e-5 * want.abs().max()).all())
    none, = (K.gated_bwd(dy, wd, gu, act, want_a=False)[1],)
    held = torch.zeros(T, 2 * Fh + 12, device="cuda")
    held[:, 4:4 + 2 * Fh] = gu
    assert none is None and torch.equal(K.gated_bwd(dy, wd, held[:, 4:4 + 2 * Fh], act)[0], dgu)
    _lib.check_status("gated")


@pytest.mark.parametrize("T,D,Fh,act", [(7, 256, 512, "silu"), (512, 512, 1024, "silu"), (1000, 256, 264, "gelu")])
def test_weight_gradients_lose_one_rounding(T, D, Fh, act):
    """Into fp32 gradients the only roundings are the operands' own, once to bf16: at most 2^-9 of a value, and so of the norm of their
    product with an operand that knows nothing of it."""
    x, w, wd, dy = make(T, D, Fh)
    w, wd = torch.nn.Parameter(w), torch.nn.Parameter(wd)
    y = F.gated_mlp(x, w, wd, act=act)
    (plain,) = torch.autograd.grad(y, wd, dy)
    a = K.gated_fwd(x, w.detach(), act)[0]
    assert torch.equal(plain, K.gemm(dy, a, a_mn_major=True, b_mn_major=True))
    w.main_grad, wd.main_grad = torch.zeros(2 * Fh, D, device="cuda"), torch.zeros(D, Fh, device="cuda")
    F.gated_mlp(x, w, wd, act=act).backward(dy)
    g, u = (x.double() @ w.detach().double().t()).chunk(2, 1)
    g.requires_grad_()
    v = ACT[act](g)
    da = dy.double() @ wd.detach().double()
    (dg,) = torch.autograd.grad(v, g, da * u)
    v = v.detach()
    for got, want in ((wd.main_grad, dy.double().t() @ (v * u)), (w.main_grad, torch.cat([dg, da * v], 1).t() @ x.double())):
        assert float((got.double() - want).norm() / want.norm()) < 2 ** -9
    assert w.grad is None and wd.grad is None


@pytest.mark.parametrize("T", [5, 200])
def test_the_same_without_the_host_module(monkeypatch, T):
    x, w, wd, dy = make(T, 64, 72)

    def run():
        t = [v.clone().requires_grad_() for v in (x, w, wd)]
        y = F.gated_mlp(*t)
        return [y.detach(), *torch.autograd.grad(y, t, dy), *K.gated_fwd(x, w, "gelu", gu_dtype=torch.float32)]

    want = run()
    monkeypatch.setattr(_lib, "host", None)
    assert all(torch.equal(a, b) for a, b in zip(want, run()))


def test_refusals():
    x, w, wd, dy = make(4, 64, 72)
    for dtype in (torch.float16, torch.float64):
        with pytest.raises(TypeError):
            K.gated_fwd(x, w, gu_dtype=dtype)
    gu = K.gated_fwd(x, w)[1]
    for bad in (gu.half(), gu.float().cpu()):
        with pytest.raises(ValueError):
            K.gated_bwd(dy, wd, bad)
