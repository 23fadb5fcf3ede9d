"""Capped scores for caps from far below the scores to far above them, in the three kernels of masked attention."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import masked_attention as MA
from tests.test_gpu_masked_attention import GRAD, OUT, close, oracle, run

pytestmark = pytest.mark.gpu

CAPS = [1e-6, 0.01, 0.5, 8.0, 30.0, 50.0, 63.0, 100.0, 300.0, 1000.0, 3000.0, 1e4, 1e5, 1e6, 1e9, 1e18]


def single(S, size, D=64, seed=0):
    """Queries and keys whose products are exact in fp32, up to about ``size`` after a scale of 1/8."""
    g = torch.Generator().manual_seed(seed + S)
    q, k = (torch.randint(-8, 9, (1, S, 2, D), generator=g).bfloat16() for _ in range(2))
    k = k * 2.0 ** round(torch.log2(torch.tensor(size / 40.0)).item())
    q[:, ::5] = 0
    return q, k


@pytest.mark.parametrize("cap", CAPS, ids=str)
@pytest.mark.parametrize("size", [0.1, 4.0, 60.0, 1000.0, 30000.0])
@pytest.mark.parametrize("kernel", ["training", "evaluation", "rows"])
def test_scores_are_capped_to_fp32(kernel, size, cap):
    """Rows that see one key have its score as their log-sum-exp."""
    S = 17 if kernel == "rows" else 300
    q, k = single(S, size)
    s = (q.double() * k.double()).sum(-1)[0].t() / 8
    want = cap * torch.tanh(s / cap)
    mask = F.attention_mask(1, S, window=1, device="cuda")
    lse = MA.masked_attention_fwd(q.cuda(), k.cuda(), k.cuda(), mask, scale=0.125, softcap=cap, for_backward=kernel == "training")[1][0].cpu().double()
    # the polynomial that scores of at most 64 in size go through has 7e-6; else the exponential and the reciprocal (2^-21 together) and a few
    # roundings of 2^-24: below 2^-19 of the score
    rel = torch.where(s.abs() <= min(cap, 64) * (1 + 1e-6), 8e-6, 2.0 ** -19)
    bad = (lse - want).abs() > rel * want.abs() + 1e-37
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, the largest error {float(((lse - want) / want).abs()[bad].max()):.1e}"
    _lib.check_status("masked attention")


@pytest.mark.parametrize("cap", [0.5, 30.0, 300.0, 1e4, 1e5, 1e6, 1e9])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("slopes", [False, True], ids=["", "slopes"])
def test_outputs_and_gradients(D, slopes, cap):
    B, S, Hq, Hkv = 2, 300, 4, 2
    g = torch.Generator().manual_seed(D)
    q, k, v, do = (torch.randn(B, S, h, D, generator=g).bfloat16() for h in (Hq, Hkv, Hkv, Hq))
    q = q * 2
    more = dict(softcap=cap, **(dict(slopes=0.05 * torch.arange(1, Hq + 1).float()) if slopes else {}))
    mask = F.attention_mask(B, S, device="cuda")
    want = oracle(q, k, v, do, mask.visible().cpu(), more)
    for name, a, b, r in zip(("out", "dq", "dk", "dv"), run(q, k, v, do, mask, more), want, (OUT, GRAD, GRAD, OUT)):
        close(a, b, r, name)
    with torch.no_grad():
        kw = {n: t.cuda() if torch.is_tensor(t) else t for n, t in more.items()}
        close(F.masked_attention(q.cuda(), k.cuda(), v.cuda(), mask, **kw), want[0], OUT, "out without a gradient")
        few = F.attention_mask(B, 3, S, device="cuda")
        close(F.masked_attention(q[:, -3:].cuda(), k.cuda(), v.cuda(), few, **kw), want[0][:, -3:], OUT, "out of few rows")
    _lib.check_status("masked attention")
