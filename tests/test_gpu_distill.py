"""Distillation kernels against the same operator on the CPU in 64 bits (held to the definition by its own tests)."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from tests.test_distill import CONFIGS, inputs

pytestmark = pytest.mark.gpu


def exact(z, labels, ids, val, gy, cfg):
    """Loss, gradient, and the sizes that their errors go by."""
    a, tau, rest = cfg.get("alpha", 1.0), cfg.get("temperature", 1.0), cfg.get("rest", False)
    loss, (logq, logq1, p, at, there, among, c, ratio, live, labelled, label) = K._distill_plain(z, labels, ids, val, a, tau, rest, -100)
    grad = K._distill_plain_grad(gy, z, labels, ids, val, a, tau, rest, -100)
    size = logq.exp() * (c + ratio)[:, None]
    size.scatter_add_(1, at, torch.where(there, p, 0.0))
    size *= a * tau
    if a < 1:
        one = logq1.exp()
        one[torch.arange(z.shape[0]), label] += 1
        size = size + (1 - a) * torch.where(labelled[:, None], one, 0.0)
    return loss, grad, size * gy.double()[:, None]


def relative(V):
    """Error of a log-sum-exp and of an exponential on it: ex2.approx 2^-22, the exponent's rounding (below 100 in size), V / 512 sums in
    a row and those of the reductions."""
    return 2 ** -22 + (100 + V / 512 + 16) * 2 ** -24


def check(z, labels, ids, val, gy, cfg, dev="cuda", threads=512):
    a, tau = cfg.get("alpha", 1.0), cfg.get("temperature", 1.0)
    want, grad, size = exact(z, labels, ids, val, gy, cfg)
    x = z.to(dev).requires_grad_(True)
    args = [None if labels is None else labels.to(dev), ids.to(dev), val.to(dev)]
    loss = F.distill_loss(x, *args, **cfg)
    (dx,) = torch.autograd.grad(loss, x, gy.to(dev))
    d = relative(z.shape[1] * 512 / threads)
    # (the teacher's weights sum to 1: an error of the log-sum-exp enters once for it and once for the label)
    assert ((loss.cpu().double() - want).abs() <= (a * tau * tau * 2 + (1 - a)) * d + 2 ** -23 * want.abs()).all()
    half = torch.finfo(z.dtype).eps / 2
    assert ((dx.cpu().double() - grad).abs() <= half * 1.01 * grad.abs() + 3 * d * size + 1e-38).all()
    # in the logits' place: the same bits
    y = z.to(dev)
    again, saved = K.distill_fwd(y, *args, **cfg)
    K.distill_bwd(gy.to(dev), y, *args, saved, out=y, **cfg)
    assert torch.equal(again, loss) and torch.equal(y, dx)
    _lib.check_status("distill")
    return loss, dx


@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,V,Kt", [(1, 1, 1), (1, 5, 2), (9, 33, 4), (8, 64, 64), (300, 1000, 31), (17, 4099, 128), (5, 32000, 700), (2, 20011, 1024)])
def test_distill(T, V, Kt, dtype, cfg):
    z, labels, ids, val, gy = inputs(T, V, Kt, cfg.get("rest", False), dtype)
    if cfg.get("rest") and Kt > V // 2:
        val = val - 0.7                                   # (something is left for the rest)
    check(z, labels, ids, val, gy, cfg)


@pytest.mark.parametrize("cfg", CONFIGS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,V,Kt", [(3100, 7, 3), (1600, 64, 8), (1000, 929, 6), (600, 4099, 128), (310, 1201, 1024), (300, 25600, 40)])
def test_many_short_rows(T, V, Kt, dtype, cfg):
    z, labels, ids, val, gy = inputs(T, V, Kt, cfg.get("rest", False), dtype)
    if cfg.get("rest") and Kt > V // 2:
        val = val - 0.7
    check(z, labels, ids, val, gy, cfg, threads=64)            # (a thread of the forward pass sums V / 64 elements)


@pytest.mark.parametrize("cfg", [CONFIGS[2], CONFIGS[5]], ids=str)
@pytest.mark.parametrize("T,V", [(1, 201088), (3, 128256), (400, 50257)])
def test_large_vocabularies(T, V, cfg):
    z, labels, ids, val, gy = inputs(T, V, 48, cfg.get("rest", False), torch.bfloat16)
    check(z, labels, ids, val, gy, cfg)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("off,pitch", [(1, 1007), (8, 1024), (3, 1003)])
def test_rows_of_a_wider_buffer(off, pitch, dtype):
    cfg = CONFIGS[2]
    z, labels, ids, val, gy = inputs(20, 1000, 8, False, dtype)
    ref = check(z, labels, ids, val, gy, cfg)
    buf = torch.full((20, pitch), 7.0, dtype=dtype, device="cuda")
    buf[:, off:off + 1000] = z.cuda()
    x = buf[:, off:off + 1000]
    args = [t.cuda() for t in (labels, ids, val)]
    loss, saved = K.distill_fwd(x, *args, **cfg)
    dx = K.distill_bwd(gy.cuda(), x, *args, saved, **cfg)
    # (a row that starts elsewhere gives its elements to other threads: sums in another order)
    assert torch.allclose(loss, ref[0], rtol=1e-5) and torch.allclose(dx.float(), ref[1].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-9)
    K.distill_bwd(gy.cuda(), x, *args, saved, out=x, **cfg)
    assert torch.equal(x, dx) and (buf[:, :off] == 7).all() and (buf[:, off + 1000:] == 7).all()
    t = z.cuda().t().contiguous().t()                      # columns apart
    assert torch.equal(K.distill_fwd(t, *args, **cfg)[0], ref[0])
    _lib.check_status("distill")


def test_types_of_ids_and_values():
    z, labels, ids, val, gy = inputs(40, 500, 9, False, torch.bfloat16)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        for it in (torch.int32, torch.int64):
            check(z, labels.to(it), ids.to(it), val.to(dt), gy, CONFIGS[2])
    check(z, None, ids.t().contiguous().t(), val.t().contiguous().t(), gy, dict(alpha=1.0, temperature=2.0))


def test_a_bad_token_stays_alone():
    """NaN or infinite logits and values of one token leave the others as they were."""
    z, labels, ids, val, gy = inputs(40, 700, 9, False, torch.bfloat16)
    ref = check(z, labels, ids, val, gy, CONFIGS[2])
    z[8, 100], z[9] = float("nan"), float("-inf")
    val[12, 3] = float("nan")
    x = z.cuda().requires_grad_(True)
    loss = F.distill_loss(x, labels.cuda(), ids.cuda(), val.cuda(), **CONFIGS[2])
    (dx,) = torch.autograd.grad(loss, x, gy.cuda())
    keep = torch.ones(40, dtype=torch.bool)
    keep[[8, 9, 12]] = False
    assert torch.equal(loss.cpu()[keep], ref[0].cpu()[keep]) and torch.equal(dx.cpu()[keep], ref[1].cpu()[keep])
    assert loss[8].isnan() and loss[12].isnan()


def test_logits_far_apart():
    """Rows whose first elements say nothing about the largest: differences that overflow a sum, and rows of -inf but for a few."""
    T, V = 12, 5003
    z, labels, ids, val, gy = inputs(T, V, 6, False, torch.float32)
    z[0, 4000] = 300.0
    z[1] -= 2000.0
    z[1, 17] = 50.0
    z[2] = float("-inf")
    z[2, 4999], z[2, 1] = 3.0, 2.0
    ids[2] = torch.tensor([4999, 1, -1, -1, -1, -1])
    labels[2] = 1
    z[3] = torch.linspace(-500, 500, V)
    z[6, ::2] = float("-inf")
    labels[6], ids[6] = 1, ids[6] // 2 * 2 + 1
    for cfg in CONFIGS:
        v = torch.log_softmax(val, 1) - 0.5 if cfg.get("rest") else val
        want, grad, size = exact(z, labels, ids, v, gy, cfg)
        x = z.cuda().requires_grad_(True)
        loss = F.distill_loss(x, labels.cuda(), ids.cuda(), v.cuda(), **cfg)
        (dx,) = torch.autograd.grad(loss, x, gy.cuda())
        a, tau = cfg.get("alpha", 1.0), cfg.get("temperature", 1.0)
        # exponents up to 2000 / ln 2 in size and the losses themselves, rounded to fp32
        d = relative(V) + 3000 / min(tau, 1.0) * 2 ** -24
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(loss.cpu()))
        assert ((loss.cpu().double() - want).abs() <= (a * tau * tau * 2 + (1 - a)) * d + 2 ** -22 * want.abs())[fine].all()
        assert ((dx.cpu().double() - grad).abs() <= 2 ** -24 * 1.01 * grad.abs() + 3 * d * size + 1e-30)[fine].all()
    _lib.check_status("distill")


def test_masked_vocabulary():
    z, labels, ids, val, gy = inputs(19, 333, 4, False, torch.bfloat16)
    z[:, 300:] = float("-inf")
    ids, labels = ids % 300, torch.where(labels >= 300, 0, labels)
    for cfg in CONFIGS:
        v = torch.log_softmax(val, 1) - 0.5 if cfg.get("rest") else val
        x = z.cuda().requires_grad_(True)
        loss = F.distill_loss(x, labels.cuda(), ids.cuda(), v.cuda(), **cfg)
        (dx,) = torch.autograd.grad(loss, x, gy.cuda())
        assert torch.isfinite(loss).all() and torch.isfinite(dx.float()).all() and (dx[:, 300:] == 0).all()


def test_captured_and_replayed_on_another_stream():
    cfg = CONFIGS[2]
    z, labels, ids, val, gy = (t.cuda() for t in inputs(64, 3001, 16, False, torch.bfloat16))
    K.distill_fwd(z, labels, ids, val, **cfg)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, saved = K.distill_fwd(z, labels, ids, val, **cfg)
        dx = K.distill_bwd(gy, z, labels, ids, val, saved, **cfg)
    for seed in (1, 2):
        z.copy_(inputs(64, 3001, 16, False, torch.bfloat16, seed)[0])
        graph.replay()
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            want, ws = K.distill_fwd(z, labels, ids, val, **cfg)
            wx = K.distill_bwd(gy, z, labels, ids, val, ws, **cfg)
            torch.cuda.current_stream().synchronize()
        assert torch.equal(loss, want) and torch.equal(dx, wx)
    _lib.check_status("distill")


@pytest.mark.parametrize("cfg", [CONFIGS[2], CONFIGS[5]], ids=str)
def test_vocabulary_projection(cfg):
    T, Dm, V = 200, 128, 1000
    _, labels, ids, val, _ = inputs(T, V, 8, cfg.get("rest", False))
    g = torch.Generator().manual_seed(3)
    x, nw, w = (torch.randn(*s, generator=g).mul(k).bfloat16() for s, k in (((T, Dm), 1), ((Dm,), 1), ((V, Dm), 0.1)))
    out = []
    for dev in ("cpu", "cuda"):
        v = [t.to(dev).requires_grad_(True) for t in (x, nw, w)]
        loss = F.lm_head_distill_loss(*v, labels.to(dev), ids.to(dev), val.to(dev), n_valid=150, **cfg)
        out.append([loss.detach().cpu()] + [t.float().cpu() for t in torch.autograd.grad(loss * 8, v)])
    # logits rounded to bf16 (2^-9 of 2, and they weigh the loss), then bf16 gradients through two products
    assert abs(out[0][0] - out[1][0]) <= 2 ** -9 * abs(out[0][0])
    for a, b in zip(out[0][1:], out[1][1:]):
        assert (a - b).norm() <= 4 * 2 ** -8 * a.norm()
    _lib.check_status("distill")
