"""MXFP4 product on the GPU: biases and residuals of other types, operands that are not what they say."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import mxfp4 as M4

pytestmark = pytest.mark.gpu


def operands(M, N, K):
    torch.manual_seed(M + N)
    q = lambda r, tile: M4.quantize(torch.randn(r, K, device="cuda").bfloat16(), row_tile=tile)[0]
    return q(M, M4.A_TILE), q(N, M4.b_tile(N))


@pytest.mark.parametrize("M,N,K", [(1, 256, 128), (7, 100, 64), (300, 520, 160)])
@pytest.mark.parametrize("which", ["bias", "residual", "both", "bf16 bias"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_bias_and_residual_keep_their_bits(M, N, K, which, out_dtype):
    """Products of 4-bit values of one block are exact in fp32; the sums over blocks and the two additions are off by less than one part
    in 2^20 of the magnitudes involved (rounded operands: one in 2^9), on top of the result's own rounding."""
    a, b = operands(M, N, K)
    bias = torch.randn(N, device="cuda") * 100
    res = torch.randn(M, N, device="cuda") * 100
    bias = None if which == "residual" else bias.bfloat16() if which == "bf16 bias" else bias
    res = None if which == "bias" else res
    got = M4.gemm(a, b, bias=bias, residual=res, out_dtype=out_dtype, alpha=0.5)
    parts = [0.5 * M4.dequantize(a).double() @ M4.dequantize(b).double().t()] + [t.double().expand(M, N) for t in (bias, res) if t is not None]
    want, size = sum(parts), 0.5 * M4.dequantize(a).double().abs() @ M4.dequantize(b).double().abs().t() + sum(p.abs() for p in parts[1:])
    limit = size * 2 ** -20 + (want.abs() * 2 ** -8 if out_dtype == torch.bfloat16 else 0)
    assert got.dtype == out_dtype and bool(((got.double() - want).abs() <= limit).all())
    if out_dtype == torch.bfloat16:
        assert torch.equal(got, M4.gemm(a, b, bias=bias, residual=res, out_dtype=torch.float32, alpha=0.5).bfloat16())
    out = torch.full((M, N), 3.0, device="cuda", dtype=out_dtype)
    M4.gemm(a, b, out=out, accumulate=True, bias=bias, residual=res, alpha=0.5)
    assert bool(((out.double() - 3 - want).abs() <= (size + 3) * 2 ** -20 + ((want + 3).abs() * 2 ** -8 if out_dtype == torch.bfloat16 else 0)).all())
    _lib.check_status("gemm")


def test_vectors_of_another_device_are_refused():
    a, b = operands(7, 256, 64)
    x, w = torch.randn(7, 64, device="cuda").bfloat16(), torch.randn(256, 64, device="cuda").bfloat16()
    for t in (dict(bias=torch.zeros(256)), dict(bias=torch.zeros(256).bfloat16()), dict(residual=torch.zeros(7, 256).bfloat16())):
        with pytest.raises(ValueError):
            M4.gemm(a, b, **t)
        with pytest.raises(ValueError):
            F.mxfp4_linear(x, w, **t)
    with pytest.raises(ValueError):
        M4.gemm(a, b, out=torch.zeros(7, 256).bfloat16())


def test_operands_that_do_not_hold_what_they_say_are_refused():
    from dataclasses import replace
    a, b = operands(7, 256, 64)
    want = M4.gemm(a, b)
    for bad in (lambda o: replace(o, rows=o.rows + 1), lambda o: replace(o, k=o.k + 128), lambda o: replace(o, sf=o.sf[:-1]),
                lambda o: replace(o, sf=o.sf.cpu()), lambda o: replace(o, q=o.q[1:])):
        for x, y in ((bad(a), b), (a, bad(b))):
            with pytest.raises(ValueError):
                M4.gemm(x, y)
        with pytest.raises(ValueError):
            M4.dequantize(bad(a))
    held = torch.zeros(7, 100, dtype=torch.uint8, device="cuda")
    held[:, 3:35] = a.q
    assert torch.equal(M4.gemm(replace(a, q=held[:, 3:35]), b), want)
    assert torch.equal(M4.dequantize(replace(a, q=held[:, 3:35])), M4.dequantize(a))
    _lib.check_status("refusals")


@pytest.mark.parametrize("T", [7, 100])
def test_gated_block_refuses_a_residual_or_weight_of_another_device(T):
    x, wgu, wd, r = (torch.randn(*s, device="cuda").bfloat16() for s in ((T, 64), (256, 64), (64, 128), (T, 64)))
    F.gated_mlp(x, wgu, wd, residual=r)
    for bad in ((x, wgu, wd, r.cpu()), (x, wgu, wd.cpu(), r), (x, wgu.cpu(), wd, r), (x, wgu, wd, r[1:])):
        with pytest.raises(ValueError):
            F.gated_mlp(*bad[:3], residual=bad[3])


def test_linear_behind_a_norm_refuses_operands_of_another_device():
    x, nw, w = torch.randn(5, 128, device="cuda").bfloat16(), torch.ones(128, device="cuda").bfloat16(), torch.randn(256, 128, device="cuda").bfloat16()
    for bad in ((x, None, nw, w.cpu()), (x, x.cpu(), nw, w), (x, None, nw.cpu(), w)):
        with pytest.raises(ValueError):
            F.add_norm_linear(*bad)
    with pytest.raises(ValueError):
        F.lm_head_loss(x, nw, w.cpu(), torch.zeros(5, dtype=torch.long, device="cuda"), precision="fp4")
