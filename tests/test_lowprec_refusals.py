"""Operands that a kernel would read at a bad address are refused before a launch.  The GPU path is walked with CPU tensors and a launcher
that only notes that it was reached."""
from dataclasses import replace

import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import kernels as K
from mlperf_training_b200.ops import mxfp4 as M4
from mlperf_training_b200.ops import mxfp8 as MX


@pytest.fixture
def launched(monkeypatch):
    """Every CPU tensor counts as one of the GPU; names of the launches."""
    names = []
    for mod in (M4, K, MX):
        monkeypatch.setattr(mod, "use_kernels", lambda t: True)
        monkeypatch.setattr(mod, "call", lambda name, *a: names.append(name))
        monkeypatch.setattr(mod, "stream_ptr", lambda: 0)
    monkeypatch.setattr(M4._lib, "gemm_workspace", lambda *a: None)
    return names


def gpu_operand(rows, k, tile):
    """As the quantiser lays it out on the GPU."""
    return M4.MX4Operand(torch.zeros(rows, k // 2, dtype=torch.uint8), torch.zeros(MX.sf_bytes(rows, k, tile), dtype=torch.uint8), rows, k, tile)


def test_product_takes_what_it_should(launched):
    a, b = gpu_operand(5, 64, M4.A_TILE), gpu_operand(40, 64, M4.b_tile(40))
    M4.gemm(a, b, bias=torch.zeros(40).bfloat16(), residual=torch.zeros(5, 40).bfloat16())
    assert launched == ["b200_gemm_mxfp4"]


@pytest.mark.parametrize("what", ["bias", "residual", "out"])
def test_product_refuses_vectors_of_another_device(launched, what):
    a, b = gpu_operand(5, 64, M4.A_TILE), gpu_operand(40, 64, M4.b_tile(40))
    t = torch.zeros(40 if what == "bias" else (5, 40), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError):
        M4.gemm(a, b, **{what: t})
    assert launched == []


BAD = {
    "short codes": lambda op: replace(op, q=op.q[:-1]),
    "wide codes": lambda op: replace(op, q=op.q[:, ::2]),
    "other codes": lambda op: replace(op, q=op.q.view(torch.int8)),
    "short scales": lambda op: replace(op, sf=op.sf[:-1]),
    "strided scales": lambda op: replace(op, sf=torch.zeros(2 * op.sf.numel(), dtype=torch.uint8)[::2]),
    "other scales": lambda op: replace(op, sf=op.sf.to(torch.int16)),
    "scales elsewhere": lambda op: replace(op, sf=op.sf.to("meta")),
    "ragged contraction": lambda op: replace(op, k=op.k - 8),
    "more rows": lambda op: replace(op, rows=op.rows + 1),
}


@pytest.mark.parametrize("why", sorted(BAD))
def test_operands_that_do_not_hold_what_they_say(launched, why):
    a, b = gpu_operand(5, 64, M4.A_TILE), gpu_operand(40, 64, M4.b_tile(40))
    for x, y in ((BAD[why](a), b), (a, BAD[why](b))):
        with pytest.raises(ValueError):
            M4.gemm(x, y)
    for op in (a, MX.MXOperand(torch.zeros(5, 64, dtype=torch.uint8), a.sf, 5, 64, 128)):
        with pytest.raises(ValueError):
            M4.dequantize(BAD[why](op))
    assert launched == []


def test_operands_of_other_layouts_are_copied(launched):
    """Rows at a larger pitch, and an address that is not a multiple of 16."""
    a, b = gpu_operand(5, 64, M4.A_TILE), gpu_operand(40, 64, M4.b_tile(40))
    wide = replace(a, q=torch.zeros(5, 100, dtype=torch.uint8)[:, 3:35])
    M4.gemm(wide, b)
    M4.dequantize(wide)
    assert launched == ["b200_gemm_mxfp4", "b200_dequant_mx"]


@pytest.mark.parametrize("T", [7, 100])
@pytest.mark.parametrize("what", ["residual", "weight", "shape"])
def test_down_projection_refuses_what_it_cannot_read(launched, T, what):
    """By the few-row kernel and by the general product alike."""
    a, w, r = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((T, 64), (128, 64), (T, 128)))
    w = w.to("meta") if what == "weight" else w
    r = r.to("meta") if what == "residual" else r[:-1] if what == "shape" else r
    with pytest.raises(ValueError):
        K.gated_down(a, w, r)
    assert launched == []


def test_linear_behind_a_norm_refuses_a_weight_of_another_device(launched):
    x, nw = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)
    for w in (torch.zeros(256, 128, dtype=torch.bfloat16, device="meta"),):
        with pytest.raises(ValueError):
            F.add_norm_linear(x, None, nw, w)
        with pytest.raises(ValueError):
            F.lm_head_loss(x, nw, w, torch.zeros(4, dtype=torch.long), precision="fp4")
    assert launched == []
