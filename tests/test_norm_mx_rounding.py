"""Both copies that the RMS norm writes are of one and the same n = (h w) rstd, rounded once."""
import pytest
import torch

from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX
from mlperf_training_b200.ops import norm_mx
from mlperf_training_b200.ops.norm_mx import rms_norm_quantize


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("T,D", [(128, 4096), (1000, 1024), (384, 8192)])
@pytest.mark.parametrize("residual", [False, True])
def test_copies_are_the_definition_bit_for_bit(dev, T, D, residual):
    torch.manual_seed(T)
    x, w = torch.randn(T, D).bfloat16().to(dev), (1 + 0.3 * torch.randn(D)).bfloat16().to(dev)
    r = torch.randn(T, D).bfloat16().to(dev) if residual else None
    row, col, h, rstd = rms_norm_quantize(x, w, residual=r, row_tile=MX.A_TILE, col_tile=MX.b_tile(D))
    n = ((h.float() * w.float()) * rstd[:, None]).cpu()          # (the product of two bf16 is exact in fp32)
    for op, v in ((row, n), (col, M4.fill_rows(n, 128).t().contiguous())):
        q, sf = norm_mx._e4m3_rows_cpu(v)
        assert torch.equal(M4.sf_plain(op).cpu(), sf) and torch.equal(op.q.cpu().view(torch.uint8), q)
