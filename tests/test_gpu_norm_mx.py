"""RMS norm with an MXFP8 output on the GPU: against 64 bits and the eager definition, the fused linear, a model that runs it with the
4-bit product and the gated block."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX
from mlperf_training_b200.ops.norm_mx import rms_norm_quantize

pytestmark = pytest.mark.gpu
EPS = 1e-5


def check_copy(op, want):
    """Half an e4m3 step of the exact value each (2^-4 of it, or half the smallest step of a scale that is at most 2 / 448 of the block's
    maximum), and 2e-6 for the sums in fp32."""
    got = M4.dequantize(op).double()
    amax = want.view(want.shape[0], -1, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(want.shape)
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= want.abs() * (2 ** -4 + 2e-6) + amax * (2 / 448 * 2 ** -10 + 1e-9)).all())
    pad = (op.k + 127) // 128 * 128
    assert int(op.sf[MX.sf_index(op.rows, pad, op.tile_rows, "cuda")][:, op.k // 32:].sum()) == 0


@pytest.mark.parametrize("T,D", [(1, 32), (1, 4096), (3, 96), (9, 1024), (127, 1056), (128, 2048), (130, 2880), (129, 4096), (257, 5120), (33, 8192),
                                 (1000, 256), (2500, 160)])
@pytest.mark.parametrize("residual", [False, True])
def test_against_64_bits(T, D, residual):
    torch.manual_seed(T + D)
    x, w = torch.randn(T, D, device="cuda").bfloat16(), (1 + 0.1 * torch.randn(D, device="cuda")).bfloat16()
    x[:, ::37] *= 20
    r = (3 * torch.randn(T, D, device="cuda")).bfloat16() if residual else None
    junk = torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda")
    del junk
    row, col, h, rstd = rms_norm_quantize(x, w, EPS, residual=r, row_tile=MX.A_TILE, col_tile=MX.b_tile(D))
    _lib.check_status("norm_mx")
    assert torch.equal(h, x if r is None else (x.float() + r.float()).bfloat16())
    hd = h.double()
    s = (hd.square().mean(1) + EPS).rsqrt()
    assert float((rstd.double() / s - 1).abs().max()) < 1e-6
    n = hd * s[:, None] * w.double()
    check_copy(row, n)
    check_copy(col, torch.cat([n, n.new_zeros(-T % 128, D)]).t().contiguous())
    for kw in (dict(row_tile=MX.A_TILE), dict(col_tile=MX.b_tile(D)), {}):
        a, b, h2, s2 = rms_norm_quantize(x, w, EPS, residual=r, **kw)
        assert (a is None or torch.equal(M4.dequantize(a), M4.dequantize(row))) and (b is None or torch.equal(M4.dequantize(b), M4.dequantize(col)))
        assert torch.equal(h2, h) and float((s2 / rstd - 1).abs().max()) < 1e-6


def test_non_finite_rows_stay_apart():
    x = torch.ones(300, 256, device="cuda").bfloat16()
    x[5, 3], x[200, 40] = float("nan"), float("inf")
    row, col, _, _ = rms_norm_quantize(x, torch.ones(256, device="cuda"), EPS, row_tile=128, col_tile=MX.b_tile(256))
    v, c = M4.dequantize(row), M4.dequantize(col).t()
    assert bool(v[5].isnan().all()) and bool(v[200, 32:64].isnan().all())
    clean = torch.ones(300, dtype=torch.bool, device="cuda")
    clean[[5, 200]] = False
    assert bool(v[clean].isfinite().all())
    assert bool(c[:32].isnan().all()) and bool(c[192:224, 40].isnan().all()) and bool(c[32:192].isfinite().all())


def test_strided_inputs_other_stream_and_no_tokens():
    torch.manual_seed(0)
    base, w = torch.randn(64, 600, device="cuda").bfloat16(), torch.randn(1200, device="cuda")[::2]
    x, r = base[:, 3:515], base[:, 80:592]
    want = rms_norm_quantize(x.clone(), w[:512].clone(), EPS, residual=r.clone(), row_tile=128, col_tile=208)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rms_norm_quantize(x, w[:512], EPS, residual=r, row_tile=128, col_tile=208)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want[:2], got[:2]):
        assert torch.equal(M4.dequantize(a), M4.dequantize(b))
    assert torch.equal(want[2], got[2]) and torch.equal(want[3], got[3])
    e = rms_norm_quantize(base[:0, :512], w[:512], EPS, row_tile=128, col_tile=208)
    assert e[0].rows == 0 and e[1].k == 0 and e[3].numel() == 0


def test_refusals():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(TypeError):
        rms_norm_quantize(x, w, EPS, row_tile=128)
    with pytest.raises(ValueError):
        rms_norm_quantize(x.bfloat16(), w.cpu(), EPS, row_tile=128)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        _lib.call("b200_norm_mx", x.data_ptr(), None, w.data_ptr(), None, w.data_ptr(), 4, 8224, EPS, None, None, 0, None, None, 0, _lib.stream_ptr())


@pytest.mark.parametrize("T,D,N", [(128, 128, 256), (256, 2048, 384), (1024, 4096, 512)])
def test_add_norm_linear(T, D, N):
    """Against the same computation in 64 bits: y and dx take one product of two 8-bit operands (each within 2^-5 of its values in the
    mean square), dw one more; the plain norm and quantiser make the same error."""
    torch.manual_seed(D)
    x, r = torch.randn(T, D, device="cuda").bfloat16().requires_grad_(), torch.randn(T, D, device="cuda").bfloat16().requires_grad_()
    nw, w = torch.ones(D, device="cuda").bfloat16().requires_grad_(), (torch.randn(N, D, device="cuda") * D ** -0.5).bfloat16().requires_grad_()
    y, h = F.add_norm_linear(x, r, nw, w, EPS)
    dy, dh = torch.randn(T, N, device="cuda").bfloat16(), torch.randn(T, D, device="cuda").bfloat16()
    dx, dr, dnw, dw = torch.autograd.grad([y, h], [x, r, nw, w], [dy, dh])
    _lib.check_status("add_norm_linear")
    assert torch.equal(dx, dr) and torch.equal(h, (x.float() + r.float()).bfloat16())
    hd, nd, wd = (t.detach().double().requires_grad_() for t in (h, nw, w))
    yd = (hd * (hd.square().mean(1, keepdim=True) + EPS).rsqrt() * nd) @ wd.t()
    ref = torch.autograd.grad([yd, hd * 1.0], [hd, nd, wd], [dy.double(), dh.double()])
    for got, want in ((y, yd), (dx, ref[0]), (dnw, ref[1]), (dw, ref[2])):
        assert float((got.double() - want).norm() / want.norm()) < 2 ** -4


def test_fp4_model_step():
    """A decoder in the recipe: the loss of the bf16 model to within what 4-bit operands allow, gradients in its direction."""
    from mlperf_training_b200.models.gpt import GPT, GPTConfig
    base = dict(n_layers=3, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn_hidden=512, vocab_size=512, seq_len=256)
    m = GPT(GPTConfig(**base, precision="fp4", bf16_last_layers=1), device="cuda")
    ref = GPT(GPTConfig(**base), device="cuda")
    ref.load_state_dict(m.state_dict())
    t = torch.randint(0, 512, (2, 257), generator=torch.Generator().manual_seed(0)).cuda()
    losses = []
    for model in (m, ref):
        loss = model(t[:, :-1], t[:, 1:])
        loss.backward()
        losses.append(float(loss))
    _lib.check_status("fp4 model")
    assert abs(losses[0] - losses[1]) < 0.02 * losses[1]
    flat = lambda model: torch.cat([p.grad.float().flatten() for p in model.parameters()])
    assert float(torch.nn.functional.cosine_similarity(flat(m), flat(ref), 0)) > 0.8
    assert getattr(m.blocks[0].w_proj, "_mx4_cache", None) is not None and getattr(m.blocks[0].w_qkv, "_mx_cache", None) is not None
