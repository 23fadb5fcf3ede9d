"""Distillation loss on the CPU: against a token-by-token definition, differences, refusals; the vocabulary projection with it."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from tests import distill_oracle as D

CONFIGS = [
    dict(alpha=1.0),
    dict(alpha=0.0),
    dict(alpha=0.7, temperature=2.0),
    dict(alpha=0.5, temperature=1.0),
    dict(alpha=1.0, temperature=0.5),
    dict(alpha=0.9, rest=True),
    dict(alpha=0.6, rest=True, temperature=3.0),
]


def inputs(T, V, Kt, rest=False, dtype=torch.float32, seed=0):
    """Logits, labels (ignored, outside and among the ids too), ids with missing entries and one twice, values."""
    g = torch.Generator().manual_seed(seed + 131 * T + V)
    z = (2 * torch.randn(T, V, generator=g)).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:Kt] if Kt <= V else torch.randint(0, V, (Kt,), generator=g) for _ in range(T)])
    val = 3 * torch.randn(T, Kt, generator=g)
    if rest:
        val = torch.log_softmax(torch.cat([val, val.amax(1, keepdim=True)], 1), 1)[:, :Kt]
    labels = torch.randint(0, V, (T,), generator=g)
    labels[::3] = ids[::3, 0]
    labels[1::5] = -100
    if T > 7:
        ids[2, 0] = -1
        ids[3, -1] = V
        val[4, 0] = float("-inf")
        ids[5] = -1                                   # no entry at all
        labels[6] = V + 3                             # no cross-entropy
        if Kt > 2 and not rest:
            ids[7, 1] = ids[7, 0]
    return z, labels, ids, val, (0.5 + torch.rand(T, generator=g)) / T


@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
@pytest.mark.parametrize("T,V,Kt", [(1, 5, 2), (9, 33, 4), (16, 100, 16), (8, 6, 6)])
def test_is_its_definition(T, V, Kt, cfg):
    z, labels, ids, val, gy = inputs(T, V, Kt, cfg.get("rest", False))
    want, grad = D.loss_and_grad(z, labels, ids, val, gy, **cfg)
    for int_type in (torch.int32, torch.int64):
        x = z.clone().requires_grad_(True)
        loss = F.distill_loss(x, labels.to(int_type), ids.to(int_type), val, **cfg)
        (dx,) = torch.autograd.grad(loss, x, gy)
        assert loss.dtype == torch.float32 and dx.dtype == z.dtype
        # one rounding to fp32 of what 64 bits give
        assert torch.allclose(loss.double(), want, rtol=2 ** -24 * 1.01, atol=1e-12)
        assert torch.allclose(dx.double(), grad, rtol=2 ** -24 * 1.01, atol=1e-14)
        out = z.clone()
        saved = K.distill_fwd(out, labels, ids, val, **cfg)[1]
        assert K.distill_bwd(gy, out, labels, ids, val, saved, out=out, **cfg) is out and torch.equal(out, dx)


@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
def test_gradient_against_differences(cfg):
    z, labels, ids, val, gy = inputs(4, 12, 3, cfg.get("rest", False))
    _, grad = D.loss_and_grad(z, labels, ids, val, gy, **cfg)
    h = 1e-5
    for t in range(4):
        for v in range(12):
            up, down = z.double().clone(), z.double().clone()
            up[t, v] += h
            down[t, v] -= h
            d = (D.loss_and_grad(up, labels, ids, val, gy, **cfg)[0] - D.loss_and_grad(down, labels, ids, val, gy, **cfg)[0]) @ gy.double() / (2 * h)
            assert abs(d - grad[t, v]) < 1e-8               # h^2 / 6 of the third derivative, 64-bit rounding over h


def test_values_that_are_the_students_own_cost_nothing():
    z, labels, ids, _, _ = inputs(9, 40, 40)
    ids = torch.arange(40).expand(9, 40).contiguous()
    loss = F.distill_loss(z.requires_grad_(True), None, ids, z.detach(), temperature=2.0)
    assert loss.abs().max() < 1e-6
    rest = F.distill_loss(z, None, ids[:, :7], torch.log_softmax(z.detach(), 1)[:, :7], rest=True)
    (dx,) = torch.autograd.grad(rest.sum(), z)
    # (log-probabilities rounded to fp32: 7 x 2^-24 x 4)
    assert rest.abs().max() < 2e-6 and dx.abs().max() < 2e-6


def test_masked_vocabulary():
    z, labels, ids, val, gy = inputs(9, 33, 4)
    z[:, 30:] = float("-inf")
    ids = ids % 30
    labels = torch.where(labels >= 30, 0, labels)
    for cfg in CONFIGS:
        v = torch.log_softmax(val, 1) - 0.5 if cfg.get("rest") else val
        x = z.clone().requires_grad_(True)
        loss = F.distill_loss(x, labels, ids, v, **cfg)
        (dx,) = torch.autograd.grad(loss, x, gy)
        assert torch.isfinite(loss).all() and torch.isfinite(dx).all() and (dx[:, 30:] == 0).all()


GOOD = dict(logits=torch.zeros(4, 9), labels=torch.zeros(4, dtype=torch.int64), ids=torch.zeros(4, 3, dtype=torch.int64), values=torch.zeros(4, 3))


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(4, 9, dtype=torch.float16)), dict(logits=torch.zeros(36)), dict(logits=torch.zeros(4, 0)), dict(labels=torch.zeros(5, dtype=torch.int64)),
    dict(labels=torch.zeros(4)), dict(ids=torch.zeros(4, 2, dtype=torch.int64)), dict(ids=torch.zeros(4, 3)), dict(ids=torch.zeros(4, 0, dtype=torch.int64), values=torch.zeros(4, 0)),
    dict(ids=torch.zeros(4, 1025, dtype=torch.int64), values=torch.zeros(4, 1025)), dict(values=torch.zeros(4, 3, dtype=torch.float64)),
    dict(values=torch.zeros(4, 3, device="meta")), dict(labels=None, alpha=0.5), dict(alpha=1.5), dict(alpha=float("nan")), dict(temperature=0.0),
    dict(temperature=float("inf")), dict(logits=torch.zeros(4, K.DISTILL_MAX_REST_V + 1, dtype=torch.bfloat16), rest=True),
])
def test_refusals(change):
    a = {**GOOD, **change}
    with pytest.raises(ValueError, match="distill"):
        F.distill_loss(a.pop("logits"), a.pop("labels"), a.pop("ids"), a.pop("values"), **a)


def test_no_tokens():
    x = torch.zeros(0, 9, requires_grad=True)
    loss = F.distill_loss(x, None, torch.zeros(0, 3, dtype=torch.int64), torch.zeros(0, 3))
    loss.sum().backward()
    assert loss.shape == (0,) and x.grad.shape == (0, 9)


@pytest.mark.parametrize("cfg", CONFIGS[2:6], ids=str)
def test_vocabulary_projection(cfg):
    T, Dm, V = 12, 16, 33
    _, labels, ids, val, _ = inputs(T, V, 4, cfg.get("rest", False))
    g = torch.Generator().manual_seed(3)
    x, nw, w = (torch.randn(*s, generator=g).requires_grad_(True) for s in ((T, Dm), (Dm,), (V, Dm)))
    loss = F.lm_head_distill_loss(x, nw, w, labels, ids, val, n_valid=5, **cfg)
    got = torch.autograd.grad(loss * 3, [x, nw, w])
    xd, nd, wd = (t.detach().double().requires_grad_(True) for t in (x, nw, w))
    z = (xd * torch.rsqrt((xd * xd).mean(-1, keepdim=True) + 1e-5) * nd) @ wd.t()
    _, dz = D.loss_and_grad(z.detach(), labels, ids, val, torch.ones(T), **cfg)
    want = torch.autograd.grad(z, [xd, nd, wd], dz * 3 / 5)
    # fp32 sums of at most 33 terms in three products in a row
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()


def test_vocabulary_projection_runs_backward_once():
    _, labels, ids, val, _ = inputs(4, 9, 2)
    x, nw, w = torch.randn(4, 8, requires_grad=True), torch.ones(8), torch.randn(9, 8)
    loss = F.lm_head_distill_loss(x, nw, w, labels, ids, val)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="second backward"):
        loss.backward()
    with torch.no_grad():
        assert torch.equal(F.lm_head_distill_loss(x, nw, w, labels, ids, val), loss.detach())
