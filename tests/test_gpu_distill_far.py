"""Distillation where a row's first columns lie far below the rest of it: finite logits at every distance at which sums taken on the largest of a
thread's first elements grow large, or are small beside those of other threads."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from tests.test_distill import inputs
from tests.test_gpu_distill import exact, relative

pytestmark = pytest.mark.gpu

FAR = [dict(alpha=1.0), dict(alpha=0.5), dict(alpha=0.7, temperature=2.0), dict(alpha=0.6, temperature=3.0), dict(alpha=0.5, temperature=8.0),
       dict(alpha=1.0, temperature=0.5), dict(alpha=0.9, rest=True), dict(alpha=0.6, rest=True, temperature=2.0)]


def far_apart(T, V, cut, dtype, cfg, by):
    """Row t: columns [0, cut) lowered by ``by[t % len(by)]``, but for the ids among them in every other row."""
    rest = cfg.get("rest", False)
    z, labels, ids, val, gy = inputs(T, V, 6, rest, torch.float32)
    low = torch.tensor(by)[torch.arange(T) % len(by)]
    keep = torch.zeros(T, V, dtype=torch.bool)
    keep[::2] = keep[::2].scatter(1, ids[::2].clamp(0, V - 1), True)
    z[:, :cut] -= torch.where(keep[:, :cut], 0.0, low[:, None])
    return z.to(dtype), labels, ids, val, gy


def check(z, labels, ids, val, gy, cfg, threads, distance, gradient=True):
    a, tau = cfg.get("alpha", 1.0), cfg.get("temperature", 1.0)
    want, grad, size = exact(z, labels, ids, val, gy, cfg)
    x = z.cuda().requires_grad_(True)
    loss = F.distill_loss(x, labels.cuda(), ids.cuda(), val.cuda(), **cfg)
    (dx,) = torch.autograd.grad(loss, x, gy.cuda())
    # beside the sums: exponents as large as the distance (in log2 units, at the temperature), rounded once each
    d = relative(z.shape[1] * 512 / threads) + 1.5 * distance / min(tau, 1.0) * 2 ** -24
    assert torch.isfinite(loss).all()
    # (a label or id that was lowered itself: the loss holds its logit, rounded)
    assert ((loss.cpu().double() - want).abs() <= (a * tau * tau * 2 + (1 - a)) * d + 2 ** -22 * want.abs()).all()
    _lib.check_status("distill")
    if not gradient:
        return
    assert torch.isfinite(dx.float()).all()
    half = torch.finfo(z.dtype).eps / 2
    assert ((dx.cpu().double() - grad).abs() <= half * 1.01 * grad.abs() + 3 * d * size + 1e-37).all()


@pytest.mark.parametrize("cfg", FAR, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,cut", [(1000, 64), (8192, 256), (8192, 2048), (8192, 4096), (32768, 4096)])
def test_first_columns_lowered(V, cut, dtype, cfg):
    by = [float(v) for v in range(60, 132, 2)] + [79.0, 83.0, 85.0, 87.0, 200.0]
    check(*far_apart(len(by), V, cut, dtype, cfg, by), cfg, 512, 200)


@pytest.mark.parametrize("cfg", FAR, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,cut", [(1000, 64), (1000, 256), (4099, 512), (4099, 2048)])
def test_many_short_rows_lowered(V, cut, dtype, cfg):
    by = [float(v) for v in range(60, 132, 2)]
    check(*far_apart(400, V, cut, dtype, cfg, by), cfg, 64, 130)


@pytest.mark.parametrize("cfg", [FAR[0], FAR[2], FAR[7]], ids=str)
def test_a_large_vocabulary_lowered(cfg):
    by = [80.0, 82.0, 84.0, 86.0, 88.0, 90.0, 92.0]
    check(*far_apart(7, 128256, 4096, torch.bfloat16, cfg, by), cfg, 512, 92)


@pytest.mark.parametrize("tau", [1.0, 2.0])
@pytest.mark.parametrize("T,V,Kt", [(5, 8192, 1024), (400, 1000, 200)])
def test_ids_far_above_all_others(T, V, Kt, tau):
    """Every thread's first elements hold an id, and ids lie 60 to 120 above the others: these are what the sum beside the ids is of."""
    cfg = dict(alpha=0.8, rest=True, temperature=tau)
    z, labels, ids, val, gy = inputs(T, V, Kt, True, torch.float32)
    ids = (torch.arange(Kt) * (V // Kt)).expand(T, Kt).contiguous()
    up = (torch.arange(60.0, 121.0, 4.0) * tau)[torch.arange(T) % 16]
    z.scatter_add_(1, ids, up[:, None].expand(T, Kt))
    check(z, labels, ids, val, gy, cfg, 64 if T > 300 else 512, 250, gradient=False)
