"""The rest of a teacher's mass where the student leaves next to nothing for it: other logits masked by a finite value."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F

CONFIGS = [dict(alpha=1.0, rest=True), dict(alpha=0.7, rest=True), dict(alpha=0.7, rest=True, temperature=2.0), dict(alpha=0.5, rest=True, temperature=8.0),
           dict(alpha=0.6, rest=True, temperature=3.0), dict(alpha=1.0, rest=True, temperature=4.0)]


def masked(T, V, Kt, low, dtype=torch.float32, seed=0):
    """Logits that are ``low`` below the rest outside the ids; labels among the ids, outside them and ignored; the teacher leaves much in some rows,
    rounding noise in others."""
    g = torch.Generator().manual_seed(seed + T + V)
    z = torch.randn(T, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:Kt] for _ in range(T)])
    among = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids, True)
    z = (z - torch.where(among, 0.0, low)).to(dtype)
    val = torch.log_softmax(torch.randn(T, Kt, generator=g), 1)
    val[::2] -= 0.3
    labels = ids[:, 0].clone()
    labels[1::3] = torch.stack([(~a).nonzero()[0, 0] for a in among])[1::3]
    labels[2::5] = -100
    return z, labels, ids, val, (0.5 + torch.rand(T, generator=g)) / T


def reference(z, labels, ids, val, gy, alpha, rest, temperature=1.0):
    """Loss and gradient in 64 bits from the definition, the log of the mass outside the ids as a log-sum-exp."""
    x, t = z.double().requires_grad_(True), val.double()
    among = torch.zeros(z.shape, dtype=torch.bool).scatter_(1, ids, True)
    logq = torch.log_softmax(x / temperature, 1)
    p = t.exp()
    r = 1 - p.sum(1)
    kl = (p * (t - logq.gather(1, ids))).sum(1)
    others = torch.logsumexp(logq.masked_fill(among, -torch.inf), 1)
    kl = kl + torch.where(r > 0, r * (r.clamp(min=1e-300).log() - others), 0.0)
    ce = -torch.log_softmax(x, 1).gather(1, labels.clamp(min=0)[:, None])[:, 0]
    loss = torch.where(labels == -100, 0.0, alpha * temperature ** 2 * kl + (1 - alpha) * ce)
    (dx,) = torch.autograd.grad((loss * gy.double()).sum(), x)
    return loss.detach(), dx


@pytest.mark.parametrize("low", [30.0, 100.0, 1e4], ids=str)
@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
def test_others_masked_by_a_finite_value(cfg, low):
    z, labels, ids, val, gy = masked(9, 40, 5, low)
    want, grad = reference(z, labels, ids, val, gy, **cfg)
    x = z.clone().requires_grad_(True)
    loss = F.distill_loss(x, labels, ids, val, **cfg)
    (dx,) = torch.autograd.grad(loss, x, gy)
    # one rounding to fp32; 64 bits hold exponents of 1e4 to 1e-12
    assert torch.allclose(loss.double(), want, rtol=2 ** -24 * 1.01, atol=1e-9)
    assert torch.allclose(dx.double(), grad, rtol=2 ** -24 * 1.01, atol=1e-10)
