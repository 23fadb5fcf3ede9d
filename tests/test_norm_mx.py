"""RMS norm with an MXFP8 output on the CPU: against 64 bits, the fused linear's gradients against formula and differences, refusals."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX
from mlperf_training_b200.ops.norm_mx import rms_norm_quantize

EPS = 1e-5


@pytest.mark.parametrize("T,D", [(1, 32), (5, 96), (128, 64), (130, 160)])
@pytest.mark.parametrize("residual", [False, True])
def test_values_against_64_bits(T, D, residual):
    """Every value is within half an e4m3 step of the exact one: 2^-4 of it, or half the smallest step (2^-10) of the block's scale,
    which is at most 2 / 448 of the block's maximum (fp32 rounding on top: 1e-6)."""
    torch.manual_seed(T + D)
    x, w = torch.randn(T, D).bfloat16(), (1 + 0.1 * torch.randn(D)).bfloat16()
    r = torch.randn(T, D).bfloat16() if residual else None
    row, col, h, rstd = rms_norm_quantize(x, w, EPS, residual=r, row_tile=128, col_tile=128)
    assert torch.equal(h, x if r is None else (x.float() + r.float()).bfloat16())
    hd = h.double()
    s = (hd.square().mean(1) + EPS).rsqrt()
    assert float((rstd.double() / s - 1).abs().max()) < 1e-6
    n = hd * s[:, None] * w.double()
    pad = torch.cat([n, n.new_zeros(-T % 128, D)])
    for op, want in ((row, n), (col, pad.t().contiguous())):
        got = M4.dequantize(op).double()
        amax = want.view(want.shape[0], -1, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(want.shape)
        assert bool(((got - want).abs() <= want.abs() * (2 ** -4 + 1e-6) + amax * (2 / 448 * 2 ** -10 + 1e-9)).all())
    assert (col.rows, col.k) == (D, (T + 127) // 128 * 128)


def test_non_finite_values_are_not_lost():
    x = torch.ones(3, 64).bfloat16()
    x[0, 3], x[1, 40] = float("nan"), float("inf")
    row, col, _, rstd = rms_norm_quantize(x, torch.ones(64), EPS, row_tile=128, col_tile=128)
    v = M4.dequantize(row)
    assert bool(v[0].isnan().all()) and float(rstd[1]) == 0.0 and bool(v[1, 32:].isnan().all()) and bool(v[2].isfinite().all())
    assert bool(M4.dequantize(col)[:, :32].isnan().all())


def test_linear_gradients():
    torch.manual_seed(2)
    T, D, N = 128, 128, 256
    x, r = torch.randn(T, D, requires_grad=True), torch.randn(T, D, requires_grad=True)
    nw, w = (1 + 0.1 * torch.randn(D)).requires_grad_(), (torch.randn(N, D) * 0.1).requires_grad_()
    y, h = F.add_norm_linear(x, r, nw, w, EPS)
    dy, dh = torch.randn(T, N), torch.randn(T, D)
    dx, dr, dnw, dw = torch.autograd.grad([y, h], [x, r, nw, w], [dy, dh])
    assert torch.equal(dx, dr)
    hd = (x + r).detach().double().requires_grad_()
    nd, wd = nw.detach().bfloat16().double().requires_grad_(), w.detach().double().requires_grad_()
    yd = (hd * (hd.square().mean(1, keepdim=True) + EPS).rsqrt() * nd) @ wd.t()
    want = torch.autograd.grad([yd, hd * 1.0], [hd, nd, wd], [dy.double(), dh.double()])
    # two operands of 8 bits in each product: 2^-5 of a value each at worst, a quarter of that in the mean
    for got, ref in zip((dx, dnw, dw), want):
        assert float((got.double() - ref).norm() / ref.norm()) < 2 ** -4
    assert float((y.double() - yd).detach().norm() / yd.detach().norm()) < 2 ** -4
    # the norm's own gradient against differences, in a direction
    v = torch.randn(T, D).double()
    f = lambda h: ((h * (h.square().mean(1, keepdim=True) + EPS).rsqrt() * nd.detach()) @ wd.detach() .t() * dy.double()).sum() + (h * dh.double()).sum()
    with torch.no_grad():
        slope = (f(hd + 1e-5 * v) - f(hd - 1e-5 * v)) / 2e-5
    assert abs(float((want[0] * v).sum() / slope) - 1) < 1e-6
    (alone,) = torch.autograd.grad(F.add_norm_linear(x, r, nw, w, EPS)[1], x, dh)
    assert torch.equal(alone, dh)


def test_no_tokens_and_refusals():
    w = torch.ones(64)
    row, col, h, rstd = rms_norm_quantize(torch.zeros(0, 64), w, EPS, row_tile=128, col_tile=128)
    assert row.rows == 0 and col.k == 0 and h.shape == (0, 64) and rstd.shape == (0,)
    x = torch.randn(4, 64)
    for bad in (lambda: rms_norm_quantize(torch.randn(4, 65), torch.ones(65)), lambda: rms_norm_quantize(torch.randn(4, 8224), torch.ones(8224)),
                lambda: rms_norm_quantize(x, torch.ones(32)), lambda: rms_norm_quantize(x, w, residual=torch.randn(3, 64)),
                lambda: rms_norm_quantize(x, w, residual=x.bfloat16()), lambda: rms_norm_quantize(x, w, row_tile=7),
                lambda: rms_norm_quantize(torch.randn(64), w), lambda: F.add_norm_linear(x, None, w, torch.randn(128, 64)),
                lambda: F.add_norm_linear(torch.randn(128, 128), None, w, torch.randn(128, 64))):
        with pytest.raises(ValueError):
            bad()


def test_fp4_model_reads_the_norm_and_trains():
    from mlperf_training_b200.models.gpt import GPT, GPTConfig
    cfg = GPTConfig(n_layers=3, hidden=128, n_heads=4, n_kv_heads=2, head_dim=32, ffn_hidden=128, vocab_size=256, seq_len=128, dtype="fp32",
                    precision="fp4", bf16_last_layers=1)
    m = GPT(cfg)
    t = torch.randint(0, 256, (1, 129), generator=torch.Generator().manual_seed(0))
    loss = m(t[:, :-1], t[:, 1:])
    loss.backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    assert getattr(m.blocks[0].w_qkv, "_mx_cache", None) is not None            # MXFP8, from the norm
    assert getattr(m.blocks[0].w_proj, "_mx4_cache", None) is not None          # 4 bits
    assert getattr(m.blocks[2].mlp.w_down, "_mx4_cache", None) is None          # the layer kept in bf16
    ref = GPT(GPTConfig(**{**cfg.to_dict(), "precision": "bf16"}))
    ref.load_state_dict(m.state_dict())
    assert abs(float(loss) - float(ref(t[:, :-1], t[:, 1:]))) < 0.05
