"""RMS norm of a residual sum with a micro-scaled output: what a block-scaled linear reads, straight from the norm.

``n = (h * weight) * rsqrt(mean(h^2) + eps)`` with ``h = x + residual`` leaves as MXFP8 operands (``ops.mxfp8``); ``n`` itself is
never written, and is rounded once, to fp32, before it is quantised (the product of two bf16 is exact there).  The backward of the norm
is ``ops.kernels.norm_bwd`` on the ``h`` and ``rstd`` that are returned here.
"""
from __future__ import annotations

import torch

from . import _lib
from . import mxfp4 as M4
from . import mxfp8 as MX
from ._lib import call, ptr, stream_ptr, use_kernels

MAX_WIDTH = 8192


def _e4m3_rows_cpu(n: torch.Tensor):
    R, C = n.shape
    sf = M4.scale_bytes(M4._amax32(n), MX.ELEMENT_FORMATS["e4m3"][2])
    inv = torch.exp2(127.0 - sf.double()).float()
    q = (n.view(R, C // 32, 32) * inv[..., None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(R, C), sf


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None,
                      row_tile: int | None = None, col_tile: int | None = None):
    """bf16 ``x [T, D]`` -> ``(row_op, col_op, h, rstd)``.

    ``h = x + residual`` rounded to bf16 (``x`` itself without a residual) is what is normalised; ``rstd [T]`` fp32.  ``row_op`` (when
    ``row_tile`` is given): rows T, contraction D.  ``col_op`` (when ``col_tile`` is given): rows D, contraction T filled up with zeros to a
    multiple of 128.  D is a multiple of 32 up to 8192; any T.  A block with an infinity or a NaN has the scale 255 (NaN)."""
    if x.is_cuda and use_kernels(x) and _lib.host is not None and row_tile != 0 and col_tile != 0:
        # (operands for inputs that are as the kernel reads them; None leaves copies and errors to the lines below)
        r = _lib.host.norm_mx(x, weight, eps, residual, row_tile or 0, col_tile or 0)
        if r is not None:
            (T, D), (q_row, sf_row, q_col, sf_col, h, rstd) = x.shape, r
            return (MX.MXOperand(q_row, sf_row, T, D, row_tile) if row_tile is not None else None,
                    MX.MXOperand(q_col, sf_col, D, (T + 127) // 128 * 128, col_tile) if col_tile is not None else None,
                    x if h is None else h, rstd)
    M4._check_matrix("rms_norm_quantize", x)
    M4._check_tile("rms_norm_quantize", row_tile)
    M4._check_tile("rms_norm_quantize", col_tile)
    T, D = x.shape
    if D > MAX_WIDTH:
        raise ValueError(f"rms_norm_quantize: {D} columns are more than {MAX_WIDTH}")
    if weight.shape != (D,):
        raise ValueError(f"rms_norm_quantize: weight {tuple(weight.shape)} for {D} columns")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"rms_norm_quantize: residual {tuple(residual.shape)} {residual.dtype} for {tuple(x.shape)} {x.dtype}")
    if any(t is not None and t.device != x.device for t in (weight, residual)):
        raise ValueError("rms_norm_quantize: operands on different devices")
    Tp = (T + 127) // 128 * 128
    if not use_kernels(x):
        h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
        hf = h.detach().float()
        rstd = torch.rsqrt((hf * hf).mean(-1) + eps)
        n = (hf * weight.detach().to(torch.bfloat16).float()) * rstd[:, None]
        row_op = MX.MXOperand(*_e4m3_rows_cpu(n), T, D, row_tile) if row_tile is not None else None
        col_op = MX.MXOperand(*_e4m3_rows_cpu(M4.fill_rows(n, 128).t().contiguous()), D, Tp, col_tile) if col_tile is not None else None
        return row_op, col_op, h, rstd
    if x.dtype != torch.bfloat16:
        raise TypeError("rms_norm_quantize: bf16 input required")
    dev = x.device
    dense = lambda t: t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
    x = dense(x)
    h = x
    if residual is not None:
        residual = dense(residual)
        h = torch.empty_like(x)
    w = dense(weight.detach().to(torch.bfloat16))
    rstd = torch.empty(T, dtype=torch.float32, device=dev)
    q_row = sf_row = q_col = sf_col = None
    if row_tile is not None:
        q_row = torch.empty((T, D), dtype=torch.uint8, device=dev)
        sf_row = torch.empty(MX.sf_bytes(T, D, row_tile), dtype=torch.uint8, device=dev)
    if col_tile is not None:
        q_col = torch.empty((D, Tp), dtype=torch.uint8, device=dev)
        sf_col = torch.empty(MX.sf_bytes(D, Tp, col_tile), dtype=torch.uint8, device=dev)
    if T:
        call("b200_norm_mx", ptr(x), ptr(residual), ptr(w), ptr(h) if residual is not None else None, ptr(rstd), T, D, float(eps), ptr(q_row),
             ptr(sf_row), row_tile or 0, ptr(q_col), ptr(sf_col), col_tile or 0, stream_ptr())
    return (MX.MXOperand(q_row, sf_row, T, D, row_tile) if row_tile is not None else None,
            MX.MXOperand(q_col, sf_col, D, Tp, col_tile) if col_tile is not None else None, h, rstd)
