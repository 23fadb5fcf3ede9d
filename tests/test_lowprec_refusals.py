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
