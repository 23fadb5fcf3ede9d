"""MXFP4 (packed e2m1 codes + one UE8M0 scale per 32 contraction elements) operands and GEMM at the 4-bit operand rate.

``quantize`` turns a bf16 matrix into the row-wise copy (contraction along the columns) and/or the column-wise copy stored
transposed (contraction along the rows, filled up with zeros to a multiple of 32), rounded to nearest or stochastically from
given bytes, the column-wise copy optionally behind the 16-row Hadamard transform; ``gemm`` multiplies two operands with
``tcgen05.mma.kind::mxf4.block_scale``; ``dequantize`` gives an operand's values (MXFP4 or MXFP8).  On CPU tensors all of it runs
as eager operations with the same rounding: the oracle of the GPU tests.

``ops.mxfp8`` carries 4-bit elements as e4m3 codes, so that one GEMM serves formats of different widths; here two elements
share a byte, which halves the operand bytes and doubles the rate of the product, for products of two 4-bit operands.

A block that holds an infinity or a NaN gets the scale 255 (NaN): the format has neither, and its 32 products are NaN.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib
from . import mxfp8 as MX
from ._lib import call, ptr, stream_ptr, use_kernels

A_TILE = 128     # M tile of the GEMM: scale-atom grouping of A operands
SF_NAN = 255


@functools.lru_cache(maxsize=1024)
def b_tile(n_rows: int) -> int:
    """N tile the GEMM uses for a B operand with ``n_rows`` rows (its scale-atom grouping)."""
    if _lib.LIB_PATH.exists():
        return int(_lib.load().b200_gemm_mxfp4_bn(int(n_rows)))     # the kernel's own rule
    return 192 if n_rows > 128 else 128


@dataclass
class MX4Operand:
    """K-major MXFP4 operand: ``q`` ``[rows, k / 2]`` bytes (element ``2 i`` in the low half of byte ``i``), ``sf`` scales.

    On CUDA ``sf`` is the flat atom layout for ``tile_rows``; on CPU a plain ``[rows, k / 32]`` uint8 matrix."""
    q: torch.Tensor
    sf: torch.Tensor
    rows: int
    k: int
    tile_rows: int

    @property
    def is_cuda(self) -> bool:
        return self.q.is_cuda


# --------------------------------------------------------------------------------------
# eager definitions
# --------------------------------------------------------------------------------------
def scale_bytes(amax: torch.Tensor, v_max: float) -> torch.Tensor:
    """Biased exponent of the smallest power of two s with ``amax / s <= v_max``; 0 for 0, at least 1 otherwise, 255 where ``amax`` is
    not finite."""
    m, e = torch.frexp(amax.double() / v_max)
    b = (torch.where(m == 0.5, e - 1, e) + 127).clamp(1, 254)
    b = torch.where(amax > 0, b, torch.zeros_like(b))
    return torch.where(torch.isfinite(amax), b, torch.full_like(b, SF_NAN)).to(torch.uint8)


def _scale_values(sf: torch.Tensor) -> torch.Tensor:
    s = torch.exp2(sf.double() - 127.0).float()
    return torch.where(sf == SF_NAN, torch.full_like(s, float("nan")), s)


def _amax32(x: torch.Tensor) -> torch.Tensor:
    """Largest magnitude per block of 32, NaN where the block holds one."""
    return x.view(x.shape[0], x.shape[1] // 32, 32).abs().amax(-1)


def _round_e2m1(y: torch.Tensor, noise: torch.Tensor | None) -> torch.Tensor:
    if noise is None:
        return MX.round_to_format(y, "e2m1")
    a = y.abs()
    quantum = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    t = torch.floor(a / quantum + (noise.float() + 0.5) / 256)
    return torch.copysign((t * quantum).clamp(max=6.0), y)


def _pack(v: torch.Tensor) -> torch.Tensor:
    """e2m1 values ``[R, C]`` to bytes ``[R, C / 2]``."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    code = torch.bucketize(v.abs(), grid).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return code[:, ::2] | (code[:, 1::2] << 4)


def _unpack(q: torch.Tensor) -> torch.Tensor:
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    code = torch.stack([q & 15, q >> 4], -1).reshape(q.shape[0], 2 * q.shape[1]).long()
    return torch.where(code >= 8, -grid[code & 7], grid[code & 7])


def _quant_rows_cpu(x: torch.Tensor, noise: torch.Tensor | None):
    R, C = x.shape
    sf = scale_bytes(_amax32(x), 6.0)
    bad = sf == SF_NAN
    inv = torch.where(bad, torch.zeros(()), torch.exp2(127.0 - sf.double()).float())
    y = torch.where(bad[..., None], torch.zeros(()), x.view(R, C // 32, 32) * inv[..., None])
    v = _round_e2m1(y, None if noise is None else noise.view(R, C // 32, 32))
    return _pack(v.view(R, C)), sf


def hadamard16(x: torch.Tensor) -> torch.Tensor:
    """Groups of 16 rows of ``x`` (fp32, a multiple of 16 rows) times the orthonormal Hadamard matrix ``(-1)^popcount(i & j) / 4``."""
    h = torch.ones(1, 1)
    while h.shape[0] < 16:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return torch.matmul(h.to(x) / 4, x.view(x.shape[0] // 16, 16, x.shape[1])).view(x.shape)


def fill_rows(x: torch.Tensor, to: int, value: float = 0) -> torch.Tensor:
    """``x`` with rows of ``value`` added up to a multiple of ``to``."""
    n = -x.shape[0] % to
    return x if n == 0 else torch.cat([x, x.new_full((n, x.shape[1]), value)])


# --------------------------------------------------------------------------------------
# operators
# --------------------------------------------------------------------------------------
def _check_matrix(what: str, x: torch.Tensor) -> None:
    if x.dim() != 2:
        raise ValueError(f"{what}: expected a 2-D tensor, got shape {tuple(x.shape)}")
    if x.shape[1] % 32 or x.shape[1] == 0:
        raise ValueError(f"{what}: {x.shape[1]} columns are not a positive multiple of 32")


def _check_tile(what: str, tile: int | None) -> None:
    if tile is not None and (tile <= 0 or tile % 16):
        raise ValueError(f"{what}: tile rows {tile} are not a positive multiple of 16")


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1] and x.data_ptr() % 16 == 0 else x.clone(
        memory_format=torch.contiguous_format)


def quantize(x: torch.Tensor, *, row_tile: int | None = None, col_tile: int | None = None, noise: torch.Tensor | None = None,
             hadamard: bool = False):
    """bf16 ``x [R, C]`` -> ``(row_op, col_op)``, C a multiple of 32, any R.

    ``row_op`` (when ``row_tile`` is given) has rows = R, contraction = C; ``col_op`` (when ``col_tile`` is given) rows = C,
    contraction = R filled up with zeros to a multiple of 32.  The tiles say how the consuming GEMM tiles the operand's rows: ``A_TILE``
    for an A operand, ``b_tile(rows)`` for a B operand.  ``noise [R, C]`` (uint8, uniform): stochastic rounding of both copies,
    element (r, c) with the byte at (r, c), 128 for the filled up rows; None: to nearest even.  ``hadamard``: the column-wise copy is that
    of the 16-row Hadamard transform of the filled up ``x``."""
    if x.is_cuda and use_kernels(x) and _lib.host is not None and row_tile != 0 and col_tile != 0:
        # (operands for an input that is as the kernel reads it; None leaves copies and errors to the lines below)
        r = _lib.host.quant_mxfp4(x, row_tile or 0, col_tile or 0, noise, hadamard)
        if r is not None:
            (R, C), (q_row, sf_row, q_col, sf_col) = x.shape, r
            return (MX4Operand(q_row, sf_row, R, C, row_tile) if row_tile is not None else None,
                    MX4Operand(q_col, sf_col, C, (R + 31) // 32 * 32, col_tile) if col_tile is not None else None)
    _check_matrix("mxfp4.quantize", x)
    _check_tile("mxfp4.quantize", row_tile)
    _check_tile("mxfp4.quantize", col_tile)
    if noise is not None and (noise.shape != x.shape or noise.dtype != torch.uint8 or noise.device != x.device):
        raise ValueError(f"mxfp4.quantize: noise {tuple(noise.shape)} {noise.dtype} on {noise.device} for an input {tuple(x.shape)} on {x.device}")
    R, C = x.shape
    Rp = (R + 31) // 32 * 32
    if not use_kernels(x):
        row_op = col_op = None
        xf = x.detach().float()
        if row_tile is not None:
            row_op = MX4Operand(*_quant_rows_cpu(xf, noise), R, C, row_tile)
        if col_tile is not None:
            v = fill_rows(xf, 32)
            v = hadamard16(v) if hadamard else v
            n = None if noise is None else fill_rows(noise, 32, 128).t().contiguous()
            col_op = MX4Operand(*_quant_rows_cpu(v.t().contiguous(), n), C, Rp, col_tile)
        return row_op, col_op
    if x.dtype != torch.bfloat16:
        raise TypeError("mxfp4.quantize: bf16 input required")
    q_row = sf_row = q_col = sf_col = None
    dev = x.device
    if row_tile is not None:
        q_row = torch.empty((R, C // 2), dtype=torch.uint8, device=dev)
        sf_row = torch.empty(MX.sf_bytes(R, C, row_tile), dtype=torch.uint8, device=dev)
    if col_tile is not None:
        q_col = torch.empty((C, Rp // 2), dtype=torch.uint8, device=dev)
        sf_col = torch.empty(MX.sf_bytes(C, Rp, col_tile), dtype=torch.uint8, device=dev)
    if R and (row_tile is not None or col_tile is not None):
        x = _aligned_rows(x)
        if noise is not None and (not noise.is_contiguous() or noise.data_ptr() % 8):
            noise = noise.clone(memory_format=torch.contiguous_format)
        call("b200_quant_mxfp4", ptr(x), x.stride(0), R, C, ptr(noise), int(hadamard), ptr(q_row), ptr(sf_row), row_tile or 0, ptr(q_col),
             ptr(sf_col), col_tile or 0, stream_ptr())
    return (MX4Operand(q_row, sf_row, R, C, row_tile) if row_tile is not None else None,
            MX4Operand(q_col, sf_col, C, Rp, col_tile) if col_tile is not None else None)


def _check_operand(what: str, op) -> None:
    """A kernel reads codes and scales by the sizes that an operand names: they have to be there."""
    per_byte = 2 if isinstance(op, MX4Operand) else 1
    if (op.rows < 0 or op.k < 0 or op.k % 32 or op.tile_rows <= 0 or op.tile_rows % 16 or op.q.dtype != torch.uint8
            or op.q.shape != (op.rows, op.k // per_byte) or op.sf.dtype != torch.uint8 or op.sf.device != op.q.device
            or not op.sf.is_contiguous() or op.sf.numel() < MX.sf_bytes(op.rows, op.k, op.tile_rows)):
        raise ValueError(f"{what}: codes {tuple(op.q.shape)} {op.q.dtype} and scales {tuple(op.sf.shape)} {op.sf.dtype} on {op.sf.device} are not "
                         f"those of {op.rows} rows of {op.k} values in tiles of {op.tile_rows} rows on {op.q.device}")


def _aligned_codes(q: torch.Tensor) -> torch.Tensor:
    return q if q.is_contiguous() and q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)


def sf_plain(op) -> torch.Tensor:
    """Scales of an MXFP4 or MXFP8 operand as a plain ``[rows, k / 32]`` uint8 matrix."""
    return op.sf if not op.is_cuda else op.sf[MX.sf_index(op.rows, op.k, op.tile_rows, op.sf.device)]


def dequantize(op, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Values ``[rows, k]`` of an MXFP4 or MXFP8 operand, as fp32 or (exactly, but for what falls below its normal numbers) bf16."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"mxfp4.dequantize: {dtype} is neither float32 nor bfloat16")
    four = isinstance(op, MX4Operand)
    if not use_kernels(op.q):
        v = _unpack(op.q) if four else op.q.view(torch.float8_e4m3fn).float()
        return (v.view(op.rows, op.k // 32, 32) * _scale_values(op.sf)[..., None]).view(op.rows, op.k).to(dtype)
    if _lib.host is not None:
        out = _lib.host.dequant_mx(op.q, op.sf, op.rows, op.k, op.tile_rows, four, dtype == torch.float32)
        if out is not None:
            return out
    _check_operand("mxfp4.dequantize", op)
    out = torch.empty((op.rows, op.k), dtype=dtype, device=op.q.device)
    if out.numel():
        call("b200_dequant_mx", ptr(_aligned_codes(op.q)), ptr(op.sf), ptr(out), op.rows, op.k, op.tile_rows, int(four), int(dtype == torch.float32),
             stream_ptr())
    return out


def _aligned_result(M: int, N: int, dtype: torch.dtype, device) -> torch.Tensor:
    """``[M, N]`` with 16-byte aligned rows."""
    per16 = 16 // dtype.itemsize
    return torch.empty((M, (N + per16 - 1) // per16 * per16), dtype=dtype, device=device)[:, :N]


def gemm(a: MX4Operand, b: MX4Operand, *, out: torch.Tensor | None = None, out_dtype=torch.bfloat16, accumulate: bool = False,
         bias: torch.Tensor | None = None, residual: torch.Tensor | None = None, alpha: float = 1.0) -> torch.Tensor:
    """``D[M,N] (+)= alpha * values(a) @ values(b)^T (+ bias[N]) (+ residual[M,N])``, bf16 or fp32.

    Any M and N.  Without ``out`` the result's rows are 16-byte aligned (for an N that is no multiple of 8 - 4 in fp32 - it is a view of
    wider rows); an ``out`` with other rows, or of such an N (the kernel's stores end on 16 bytes), is filled through one like that.  An empty
    contraction gives the bias and the residual alone.  A bias or a residual with more bits than bf16 is added in fp32."""
    if not isinstance(a, MX4Operand) or not isinstance(b, MX4Operand):
        raise TypeError("mxfp4.gemm: both operands must be MXFP4")
    if a.k != b.k:
        raise ValueError(f"mxfp4.gemm: contraction mismatch {a.k} vs {b.k}")
    for t in (b.q, out, bias, residual):
        if t is not None and t.device != a.q.device:
            raise ValueError(f"mxfp4.gemm: operands on {a.q.device} and {t.device}")
    M, N, Kd = a.rows, b.rows, a.k
    if out is not None:
        if out.shape != (M, N):
            raise ValueError(f"mxfp4.gemm: bad output {tuple(out.shape)} for {M}x{N}")
        out_dtype = out.dtype
    elif accumulate:
        raise ValueError("mxfp4.gemm: accumulate needs an output tensor")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"mxfp4.gemm: bias {tuple(bias.shape)} for {N} columns")
    if residual is not None and residual.shape != (M, N):
        raise ValueError(f"mxfp4.gemm: residual {tuple(residual.shape)} for {M}x{N}")
    if not use_kernels(a.q) or Kd == 0:
        d = alpha * (dequantize(a) @ dequantize(b).t())
        d = d if bias is None else d + bias.float()
        d = d if residual is None else d + residual.float()
        if out is None:
            return d.to(out_dtype)
        return out.add_(d.to(out.dtype)) if accumulate else out.copy_(d.to(out.dtype))
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("mxfp4.gemm: output must be bf16 or fp32")
    if a.tile_rows != A_TILE or b.tile_rows != b_tile(N):
        raise ValueError(f"mxfp4.gemm: operand scale tiling ({a.tile_rows}, {b.tile_rows}) does not match the kernel tiles ({A_TILE}, {b_tile(N)})")
    if (bias is not None and bias.dtype != torch.bfloat16) or (residual is not None and residual.dtype != torch.bfloat16):
        # (the kernel's epilogue adds bf16; what has more bits is added to the fp32 product here, and the sum rounded once)
        d = gemm(a, b, out_dtype=torch.float32, bias=bias if bias is not None and bias.dtype == torch.bfloat16 else None,
                 residual=residual if residual is not None and residual.dtype == torch.bfloat16 else None, alpha=alpha)
        for t in (bias, residual):
            if t is not None and t.dtype != torch.bfloat16:
                d = d.add_(t.float())
        if out is None:
            return d if out_dtype == torch.float32 else _aligned_result(M, N, out_dtype, d.device).copy_(d)
        return out.copy_(d.add_(out) if accumulate else d)
    if out is None and _lib.host is not None:
        d = _lib.host.gemm_mxfp4(a.q, a.sf, a.tile_rows, b.q, b.sf, b.tile_rows, M, N, Kd, out_dtype == torch.float32, bias, residual, alpha)
        if d is not None:
            return d
    _check_operand("mxfp4.gemm", a)
    _check_operand("mxfp4.gemm", b)
    if out is not None and (out.stride(1) != 1 or (N * out.element_size()) % 16 or (out.stride(0) * out.element_size()) % 16 or out.data_ptr() % 16 or out.stride(0) < N):
        if M and N:
            d = gemm(a, b, out_dtype=torch.float32 if accumulate else out_dtype, bias=bias, residual=residual, alpha=alpha)
            out.copy_(out.float().add_(d)) if accumulate else out.copy_(d)
        return out
    if out is None:
        out = _aligned_result(M, N, out_dtype, a.q.device)
    if M == 0 or N == 0:
        return out
    if bias is not None:
        bias = bias.contiguous()
    ldr = 0
    if residual is not None:
        if residual.stride(1) != 1:
            residual = residual.contiguous()
        ldr = residual.stride(0)
    ws = _lib.gemm_workspace("b200_gemm_mxfp4_workspace", M, N, Kd, a.q.device)
    a_q, b_q = _aligned_codes(a.q), _aligned_codes(b.q)
    call("b200_gemm_mxfp4", ptr(a_q), ptr(a.sf), ptr(b_q), ptr(b.sf), ptr(out), M, N, Kd, a_q.stride(0), b_q.stride(0), out.stride(0),
         int(out.dtype == torch.float32), int(accumulate), ptr(bias), ptr(residual), ldr, float(alpha), ptr(ws),
         0 if ws is None else ws.numel(), stream_ptr())
    return out
