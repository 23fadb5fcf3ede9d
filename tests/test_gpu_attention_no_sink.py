"""Sink logits of -inf are no sink: rows that see nothing have no gradient of it."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Sq", [200, 700])
def test_a_sink_that_is_not_there(Sq):
    B, H, D = 2, 4, 64
    g = torch.Generator().manual_seed(Sq)
    q, k, v, do = (torch.randn(B, Sq, H, D, generator=g).bfloat16().cuda() for _ in range(4))
    ids = torch.zeros(B, Sq, dtype=torch.int32, device="cuda")
    ids[:, 50:80] = -1
    mask = F.attention_mask(B, Sq, documents=ids)
    sink = torch.tensor([0.3, -torch.inf, 0.1, -torch.inf], device="cuda")
    out = []
    for t in (sink, torch.where(sink == -torch.inf, -1e4, sink)):
        ins = [x.clone().requires_grad_(True) for x in (q, k, v, t)]
        y = F.masked_attention(*ins[:3], mask, sink=ins[3])
        out.append([y] + list(torch.autograd.grad(y, ins, do)))
    # a logit of -1e4 has no weight either in rows that see something
    seen = ids >= 0
    assert torch.equal(out[0][0][seen], out[1][0][seen])
    assert torch.isfinite(out[0][4]).all() and (out[0][4][1::2] == 0).all()
    assert torch.allclose(out[0][4], out[1][4], rtol=1e-5, atol=1e-6)
    assert all(torch.isfinite(t.float()).all() for t in out[0])
    _lib.check_status("masked attention")
