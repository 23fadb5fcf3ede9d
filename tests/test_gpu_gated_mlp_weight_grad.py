"""Gradient of the gated block's down projection on the GPU: from the activation that the forward multiplied."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,Fh,act", [(7, 256, 512, "silu"), (512, 512, 1024, "silu"), (1000, 256, 264, "gelu")])
def test_down_projection_gradient_reads_the_forwards_activation(T, D, Fh, act):
    """Into an fp32 gradient the only rounding is the activation's own, once to bf16: at most 2^-9 of a value, and so of the norm of its
    product with a gradient that knows nothing of it (made again from the rounded projections it has two roundings more)."""
    torch.manual_seed(T)
    x = torch.randn(T, D, device="cuda").bfloat16()
    w, wd = torch.nn.Parameter((torch.randn(2 * Fh, D, device="cuda") * D ** -0.5).bfloat16()), torch.nn.Parameter((torch.randn(D, Fh, device="cuda") * 0.05).bfloat16())
    dy = torch.randn(T, D, device="cuda").bfloat16()
    y = F.gated_mlp(x, w, wd, act=act)
    (plain,) = torch.autograd.grad(y, wd, dy)
    a = K.gated_fwd(x, w.detach(), act)[0]
    assert torch.equal(plain, K.gemm(dy, a, a_mn_major=True, b_mn_major=True))
    wd.main_grad = torch.zeros(D, Fh, device="cuda")
    F.gated_mlp(x, w, wd, act=act).backward(dy)
    g, u = (x.double() @ w.detach().double().t()).chunk(2, 1)
    v = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    want = dy.double().t() @ (v * u)
    assert wd.grad is None and float((wd.main_grad.double() - want).norm() / want.norm()) < 2 ** -9


def test_frozen_down_projection_keeps_no_activation():
    x = torch.randn(64, 64, device="cuda").bfloat16().requires_grad_()
    w, wd = torch.randn(256, 64, device="cuda").bfloat16(), torch.randn(64, 128, device="cuda").bfloat16()
    held = lambda y: sum(t.numel() for t in y.grad_fn.saved_tensors if t is not None)
    frozen, trained = held(F.gated_mlp(x, w, wd)), held(F.gated_mlp(x, w, wd.clone().requires_grad_()))
    assert trained - frozen == 64 * 128
