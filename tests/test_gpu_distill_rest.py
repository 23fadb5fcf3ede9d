"""Distillation with the teacher's rest as an event of its own, where the student leaves next to nothing outside the teacher's ids."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from tests.test_distill_rest import CONFIGS, masked, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [30.0, 80.0, 88.0, 100.0, 300.0, 1e4], ids=str)
@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,V,Kt", [(6, 50, 7), (3, 9001, 33), (400, 700, 12)])
def test_others_masked_by_a_finite_value(T, V, Kt, dtype, cfg, low):
    z, labels, ids, val, gy = masked(T, V, Kt, low, dtype)
    want, grad = reference(z, labels, ids, val, gy, **cfg)
    x = z.cuda().requires_grad_(True)
    loss = F.distill_loss(x, labels.cuda(), ids.cuda(), val.cuda(), **cfg)
    (dx,) = torch.autograd.grad(loss, x, gy.cuda())
    a, tau = cfg["alpha"], cfg.get("temperature", 1.0)
    # exponents of at most 1.5 low / tau + 30 log2 units, differences of such log-sum-exps, V / 64 sums in a row: of a term's size, which is 2 at most
    d = (1.5 * low / tau + 130 + V / 64) * 2 ** -24 + 2 ** -21
    assert torch.isfinite(dx.float()).all() and torch.isfinite(loss).all()
    # (the loss holds r times the distance between the log-sum-exps, each rounded to fp32, and the label's logit)
    assert ((loss.cpu().double() - want).abs() <= 3 * (a * tau * tau + 1) * d + 2 ** -22 * want.abs()).all()
    half = torch.finfo(dtype).eps / 2
    assert ((dx.cpu().double() - grad).abs() <= half * 1.01 * grad.abs() + 4 * d * gy.double()[:, None] * (a * tau + 1)).all()
    y = z.cuda()
    again, saved = K.distill_fwd(y, labels.cuda(), ids.cuda(), val.cuda(), **cfg)
    K.distill_bwd(gy.cuda(), y, labels.cuda(), ids.cuda(), val.cuda(), saved, out=y, **cfg)
    assert torch.equal(again, loss) and torch.equal(y, dx)
    _lib.check_status("distill")
