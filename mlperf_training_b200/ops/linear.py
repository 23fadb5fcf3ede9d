"""Precision-aware GEMM triple of a linear layer (forward, dgrad, wgrad).

``precision="bf16"`` runs the bf16 tcgen05 GEMM on the tensors as they are (the backward GEMMs read
the same row-major buffers as MN-major operands).  ``precision="fp8"`` runs the per-tensor FP8 GEMM
(e4m3 activations and weights, e5m2 gradients, delayed scaling: ``ops.fp8``); the scale state of the
three tensor sites of a linear (input, weight, output gradient) lives on the weight parameter.
``precision="mxfp8"`` runs the block-scaled
GEMM: activations and gradients are quantised on the fly (one pass gives the row-wise copy for the
next GEMM and the transposed column-wise copy that the weight-gradient GEMM needs later), weights
are quantised once per optimizer step in both directions and cached on the parameter.  The narrower
members of the micro-scaled family (``mxfp6``, ``mxfp4``, ``a6w4``: ``MX_RECIPES``) run the same GEMM on
operands whose elements were rounded to the 6- or 4-bit format first - every such value is an e4m3 value, so
the product is the narrow format's, bit for bit, at the 8-bit operand rate; gradients of the 4-bit recipes are
rounded stochastically and their weight-gradient operands pass a block Hadamard transform along the tokens.

``precision="fp4"`` runs the product itself on 4-bit operands (``ops.mxfp4``): activations and weights rounded to nearest, output
gradients stochastically, both operands of the weight gradient behind a 16-row Hadamard transform.

What is saved for backward is the return value of ``forward`` (a bf16 tensor or the fp8 operand);
``Saved.pack`` / ``Saved.unpack`` move it through ``ctx.save_for_backward``.

Mirrors the recipe plumbing the reference gets from Transformer Engine (quantised copies of
weights cached between micro-batches, column-wise copies kept for wgrad;
llama2_sft/primus/src/llama2_custom.py:1904-1910 pre-quantises frozen base weights once).
"""
from __future__ import annotations

import torch
from torch.multiprocessing.reductions import StorageWeakRef

from . import fp8 as F8
from . import kernels as K
from . import mxfp4 as M4
from . import mxfp8 as MX
from ._lib import stream_ptr

# bumped by the optimizer engine after every parameter update: invalidates cached weight copies
_WEIGHT_EPOCH = 0


def weight_epoch() -> int:
    """Counter that advances whenever parameters may have changed outside autograd's version tracking."""
    return _WEIGHT_EPOCH


def bump_weight_epoch() -> None:
    global _WEIGHT_EPOCH
    _WEIGHT_EPOCH += 1


# micro-scaled recipes: element format of (forward activation, forward weight, gradient, backward weight, activation kept
# for the weight gradient), stochastic rounding of the gradient operands, Hadamard block along the tokens for the
# weight-gradient operands (0 = none).  "a6w4": forward in MXFP6 activations x MXFP4 weights, backward in MXFP4
# (flux1/primus/patches/flux_fprop_switch.py:36-120); "mxfp4": llama2_sft/primus/patches/megatron_lm_mxfp4_recipe.patch:66-84.
MX_RECIPES = {
    "mxfp8": ("e4m3", "e4m3", "e4m3", "e4m3", "e4m3", False, 0),
    "mxfp6": ("e2m3", "e2m3", "e3m2", "e2m3", "e2m3", False, 0),
    "mxfp4": ("e2m1", "e2m1", "e2m1", "e2m1", "e2m1", True, 16),
    "a6w4": ("e2m3", "e2m1", "e2m1", "e2m1", "e2m1", True, 16),
    # the phase a FLUX run switches to: forward at 8 bits, backward still at 4
    "mxfp8_fwd_mxfp4_bwd": ("e4m3", "e4m3", "e2m1", "e2m1", "e2m1", True, 16),
}


def weight_format(precision: str) -> str:
    """Element format of the forward weights of a micro-scaled recipe (e4m3 for every other precision); "fp4": of those it multiplies in 4 bits."""
    return "e2m1" if precision == "fp4" else MX_RECIPES.get(precision, ("", "e4m3"))[1]


def is_mx(precision: str) -> bool:
    return precision in MX_RECIPES


_HADAMARD: dict = {}


def hadamard_rows(x: torch.Tensor, block: int) -> torch.Tensor:
    """``x [T, C]`` with every group of ``block`` consecutive rows multiplied by the orthonormal Hadamard matrix of that
    size: ``hadamard_rows(a).T @ hadamard_rows(b) == a.T @ b`` exactly in real arithmetic, while outliers of a column are
    spread over the block before the operands are rounded."""
    key = (block, x.device, x.dtype)
    h = _HADAMARD.get(key)
    if h is None:
        h = torch.ones(1, 1)
        while h.shape[0] < block:
            h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
        h = _HADAMARD[key] = (h / block ** 0.5).to(device=x.device, dtype=x.dtype)
    T, C = x.shape
    return torch.matmul(h, x.reshape(T // block, block, C)).reshape(T, C)


def mx_eligible(rows: int, n_out: int, n_in: int) -> bool:
    """MXFP8 needs every GEMM dimension to be a multiple of 128 (tokens, out and in features)."""
    return rows % 128 == 0 and n_out % 128 == 0 and n_in % 128 == 0


def _identity(weight: torch.Tensor):
    """What a change of ``weight`` through torch alters: the version that in-place operations count up, storage, address, type, layout.
    (The reference names the storage for good and does not keep its memory; an address may come back with another one.)"""
    return weight._version, StorageWeakRef(weight.untyped_storage()), weight.data_ptr(), weight.dtype, weight.shape, weight.stride()


def _is_still(weight: torch.Tensor, identity) -> bool:
    version, storage, address, dtype, shape, stride = identity
    return (weight._version == version and weight.untyped_storage()._cdata == storage.cdata and weight.data_ptr() == address
            and weight.dtype is dtype and weight.shape == shape and weight.stride() == stride)


def _epoch(weight: torch.Tensor) -> int:
    return _WEIGHT_EPOCH if weight.requires_grad else -1


def _kept_copies(weight: torch.Tensor, slot: str, formats: tuple, need_col: bool, make):
    """(row, col) copies of ``weight [N, K]`` for forward and dgrad, kept on the tensor under ``slot`` until it changes: through torch (in
    place, or with other storage) or through an optimizer step.  What torch does not see - writes through ``weight.data``, or by a kernel -
    has to be followed by ``bump_weight_epoch()``.  ``make(w, formats, need_row, need_col)``: the copies asked for;
    ``formats``: what besides the weight they depend on.

    A call on another stream than the one that made them waits for them there.  A call under graph capture makes its own, inside the
    graph: what it records is not made yet when it returns, copies made outside the graph may be gone when it is replayed, and a replay
    follows the weight as it does with any tensor.  Of tensors made in inference mode, whose updates torch does not count, none are kept.

    An entry: ((epoch, *formats), row, col, identity of the weight, stream, event behind the making)."""
    keep = not weight.is_inference() and not (weight.is_cuda and torch.cuda.is_current_stream_capturing())
    row = None
    if keep:
        key = (_epoch(weight), *formats)
        cache = getattr(weight, slot, None)
        if cache is not None and cache[0] == key and _is_still(weight, cache[3]):
            if cache[4] is not None and cache[4] != stream_ptr():
                _use_here(cache)
            if cache[2] is not None or not need_col:
                return cache[1], cache[2]
            row = cache[1]               # (a forward that expected no backward left it: only the other copy is missing)
    w = weight.detach()
    if w.dtype != torch.bfloat16 and w.is_cuda:
        w = w.to(torch.bfloat16)
    new_row, col = make(w, formats, row is None, need_col)
    row = new_row if row is None else row
    if keep:
        stream = event = None
        if w.is_cuda:
            # (torch.cuda.current_stream(), which record() would call, takes several Python layers)
            i, d, t = torch._C._cuda_getCurrentStream(torch._C._cuda_getDevice())
            stream, event = stream_ptr(), torch.cuda.Event()
            event.record(torch.cuda.Stream(stream_id=i, device_index=d, device_type=t))
        setattr(weight, slot, (key, row, col, _identity(weight), stream, event))
    return row, col


def _use_here(cache) -> None:
    """Order the current stream behind the making of kept copies, and keep their memory until it is done with them."""
    here = torch.cuda.current_stream()
    here.wait_event(cache[5])
    for op in cache[1:3]:
        if op is not None:
            op.q.record_stream(here)
            op.sf.record_stream(here)


def copies_kept(weight: torch.Tensor, slot: str, need_col: bool) -> bool:
    """Whether the copies under ``slot`` are those of the weight as it is now (in whatever format they were made)."""
    cache = getattr(weight, slot, None)
    return (cache is not None and cache[0][0] == _epoch(weight) and (cache[2] is not None or not need_col)
            and not weight.is_inference() and _is_still(weight, cache[3]))


def _make_mx(w: torch.Tensor, formats: tuple, need_row: bool, need_col: bool):
    N, Kd = w.shape
    return MX.quantize(w, row_tile=MX.b_tile(N) if need_row else None, col_tile=MX.b_tile(Kd) if need_col else None, fmt=formats[0],
                       col_fmt=formats[1])


def weight_operands(weight: torch.Tensor, need_col: bool = True, fmt: str = "e4m3", col_fmt: str | None = None):
    """(w_row, w_col) micro-scaled copies of ``weight`` ``[N, K]``: ``w_row`` (rows N, contraction K) is
    the B operand of forward, ``w_col`` (rows K, contraction N) the B operand of dgrad; ``fmt`` / ``col_fmt``: their element
    formats.  Kept on the tensor by the rules of ``_kept_copies``."""
    return _kept_copies(weight, "_mx_cache", (fmt, col_fmt or fmt), need_col, _make_mx)


def _site(weight: torch.Tensor, name: str, fmt: str) -> "F8.DelayedScale":
    """Delayed-scaling state of one tensor site of the linear that owns ``weight``."""
    sites = getattr(weight, "_fp8_sites", None)
    if sites is None:
        sites = weight._fp8_sites = {}
    st = sites.get(name)
    if st is None or st.fmt != fmt:
        st = sites[name] = F8.DelayedScale(fmt, weight.device)
    return st


def fp8_weight_operands(weight: torch.Tensor, need_col: bool = True):
    """(w_row, w_col) per-tensor e4m3 copies of ``weight [N, K]`` (``w_col`` is the transposed copy for
    dgrad), cached until the next optimizer step."""
    cache = getattr(weight, "_fp8_cache", None)
    epoch = _WEIGHT_EPOCH if weight.requires_grad else -1
    if cache is not None and cache[0] == epoch and (cache[2] is not None or not need_col):
        return cache[1], cache[2]
    w = weight.detach()
    if w.dtype != torch.bfloat16 and w.is_cuda:
        w = w.to(torch.bfloat16)
    st = _site(weight, "w", "e4m3")
    st.prepare(w, epoch)
    row, col = F8.quantize(w, st, want_row=True, want_col=need_col)
    weight._fp8_cache = (epoch, row, col)
    return row, col


def fp4_eligible(rows: int, n_out: int, n_in: int) -> bool:
    """The 4-bit product contracts over whole blocks of 32: output features in dgrad, input features in forward (tokens are filled up)."""
    return rows > 0 and n_out > 0 and n_in > 0 and n_out % 32 == 0 and n_in % 32 == 0


def _make_mx4(w: torch.Tensor, formats: tuple, need_row: bool, need_col: bool):
    N, Kd = w.shape
    return M4.quantize(w, row_tile=M4.b_tile(N) if need_row else None, col_tile=M4.b_tile(Kd) if need_col else None)


def fp4_weight_operands(weight: torch.Tensor, need_col: bool = True):
    """(w_row, w_col) MXFP4 copies of ``weight [N, K]`` for forward and dgrad, kept on the tensor by the rules of ``_kept_copies``."""
    return _kept_copies(weight, "_mx4_cache", (), need_col, _make_mx4)


def fp4_forward(x: torch.Tensor, weight: torch.Tensor, *, bias=None, residual=None, need_wgrad: bool = True, need_dgrad: bool = False):
    """``y = Q(x) Q(W)^T (+ bias) (+ residual)``; returns ``(y, saved)``, ``saved`` the column-wise copy of the Hadamard transform of ``x``."""
    w_row, _ = fp4_weight_operands(weight, need_col=need_dgrad)
    xq = x if x.dtype == torch.bfloat16 or not x.is_cuda else x.to(torch.bfloat16)
    x_row, x_col = M4.quantize(xq, row_tile=M4.A_TILE, col_tile=M4.b_tile(x.shape[1]) if need_wgrad else None, hadamard=True)
    return M4.gemm(x_row, w_row, bias=bias, residual=residual, out_dtype=x.dtype), x_col


def fp4_backward(dy: torch.Tensor, saved, weight: torch.Tensor, *, noise: torch.Tensor | None = None, need_dx: bool = True,
                 need_dw: bool = True):
    """``(dx, dw)``: ``dx = Qs(dy) Q(W^T)^T``, ``dw = Qs(H dy)^T Q(H x)`` (None when it went into ``weight.main_grad``).  ``noise``: the bytes of
    the stochastic rounding, one per element of ``dy``; None: drawn here."""
    dx = dw = None
    if not (need_dx or need_dw):
        return dx, dw
    dyq = dy if dy.dtype == torch.bfloat16 or not dy.is_cuda else dy.to(torch.bfloat16)
    if noise is None:
        noise = torch.randint(0, 256, dy.shape, dtype=torch.uint8, device=dy.device)
    dy_row, dy_col = M4.quantize(dyq, row_tile=M4.A_TILE if need_dx else None, col_tile=M4.A_TILE if need_dw else None, noise=noise,
                                 hadamard=True)
    if need_dx:
        _, w_col = fp4_weight_operands(weight, need_col=True)
        dx = M4.gemm(dy_row, w_col, out_dtype=dy.dtype)
    if need_dw:
        if not isinstance(saved, M4.MX4Operand):         # (a forward of another precision left its activation as it was)
            _, saved = M4.quantize(saved, col_tile=M4.b_tile(weight.shape[1]), hadamard=True)
        mg = getattr(weight, "main_grad", None)
        if mg is not None:
            M4.gemm(dy_col, saved, out=mg, accumulate=True)
        else:
            dw = M4.gemm(dy_col, saved, out_dtype=weight.dtype)
    return dx, dw


class Saved:
    """The activation copy kept for the weight-gradient GEMM."""

    @staticmethod
    def pack(obj):
        if isinstance(obj, MX.MXOperand):
            return [obj.q, obj.sf], ("mx", obj.rows, obj.k, obj.tile_rows)
        if isinstance(obj, M4.MX4Operand):
            return [obj.q, obj.sf], ("mx4", obj.rows, obj.k, obj.tile_rows)
        if isinstance(obj, F8.FP8Operand):
            return [obj.q, obj.inv_scale], ("f8", obj.rows, obj.k, obj.fmt)
        return [obj], ("t",)

    @staticmethod
    def unpack(tensors, meta):
        if meta[0] == "mx":
            return MX.MXOperand(tensors[0], tensors[1], meta[1], meta[2], meta[3])
        if meta[0] == "mx4":
            return M4.MX4Operand(tensors[0], tensors[1], meta[1], meta[2], meta[3])
        if meta[0] == "f8":
            return F8.FP8Operand(tensors[0], tensors[1], meta[1], meta[2], meta[3])
        return tensors[0]


def low_precision(precision: str, rows: int, n_out: int, n_in: int) -> bool:
    """The call runs a quantised GEMM (and saves a quantised activation copy for backward)."""
    if precision == "fp4":
        return fp4_eligible(rows, n_out, n_in)
    # (the per-tensor FP8 GEMM has CTA-pair tiles only: its M - the tokens in forward and dgrad, the output
    # features in wgrad - must exceed one 128-row tile)
    return (is_mx(precision) or precision == "fp8") and mx_eligible(rows, n_out, n_in) and (is_mx(precision) or (rows > 128 and n_out > 128))


def forward(x: torch.Tensor, weight: torch.Tensor, precision: str, *, bias=None, residual=None,
            need_wgrad: bool = True, need_dgrad: bool = False):
    """``y = x W^T (+ bias) (+ residual)``.  Returns ``(y, saved)`` where ``saved`` is what
    ``backward`` needs of ``x`` (None when ``need_wgrad`` is False).  ``need_dgrad``: the backward will ask for ``dx``, so the
    micro-scaled copies of the weight for both directions are made in one pass over it."""
    M, Kd = x.shape
    N = weight.shape[0]
    if is_mx(precision) and mx_eligible(M, N, Kd):
        f_act, f_w, _, b_w, b_act, _, had = MX_RECIPES[precision]
        w_row, _ = weight_operands(weight, need_col=need_dgrad, fmt=f_w, col_fmt=b_w)
        if had and need_wgrad and M % had == 0:
            # the copy kept for the weight gradient passes the Hadamard transform along the tokens (its partner, the
            # output gradient, gets the same one in backward)
            x_row, _ = MX.quantize(x, row_tile=MX.A_TILE, fmt=f_act)
            _, x_col = MX.quantize(hadamard_rows(x, had), col_tile=MX.b_tile(Kd), fmt=b_act)
        else:
            x_row, x_col = MX.quantize(x, row_tile=MX.A_TILE, col_tile=MX.b_tile(Kd) if need_wgrad else None, fmt=f_act,
                                       col_fmt=b_act)
        y = MX.gemm(x_row, w_row, bias=bias, residual=residual, out_dtype=x.dtype)
        return y, x_col
    if precision == "fp4" and fp4_eligible(M, N, Kd):
        return fp4_forward(x, weight, bias=bias, residual=residual, need_wgrad=need_wgrad, need_dgrad=need_dgrad)
    if precision == "fp8" and low_precision(precision, M, N, Kd):
        w_row, _ = fp8_weight_operands(weight, need_col=False)
        st = _site(weight, "x", "e4m3")
        st.prepare(x, _WEIGHT_EPOCH)
        x_row, x_col = F8.quantize(x, st, want_row=True, want_col=need_wgrad)
        y = F8.gemm(x_row, w_row, bias=bias, residual=residual, out_dtype=x.dtype)
        return y, x_col
    y = K.gemm(x, weight, bias=bias, residual=residual)
    return y, (x if need_wgrad else None)


def backward(dy: torch.Tensor, saved, weight: torch.Tensor, precision: str, *, need_dx: bool = True,
             need_dw: bool = True):
    """Returns ``(dx, dw)``.  ``dw`` is None when it was accumulated into ``weight.main_grad``
    (or not requested)."""
    M, N = dy.shape
    Kd = weight.shape[1]
    dx = dw = None
    use_mx = is_mx(precision) and mx_eligible(M, N, Kd)
    if use_mx:
        _, f_w, g_fmt, b_w, b_act, g_sr, had = MX_RECIPES[precision]
        had = had if M % max(had, 1) == 0 else 0
    if use_mx and need_dw and not isinstance(saved, MX.MXOperand):
        # the forward ran in bf16 for this call (e.g. recomputed activation): quantise now
        _, saved = MX.quantize(hadamard_rows(saved, had) if had else saved, col_tile=MX.b_tile(Kd), fmt=b_act)
    if use_mx:
        if had and need_dw:
            dy_row = MX.quantize(dy, row_tile=MX.A_TILE, fmt=g_fmt, stochastic=g_sr)[0] if need_dx else None
            _, dy_col = MX.quantize(hadamard_rows(dy, had), col_tile=MX.A_TILE, fmt=g_fmt, stochastic=g_sr)
        else:
            dy_row, dy_col = MX.quantize(dy, row_tile=MX.A_TILE if need_dx else None,
                                         col_tile=MX.A_TILE if need_dw else None, fmt=g_fmt, stochastic=g_sr)
        if need_dx:
            _, w_col = weight_operands(weight, need_col=True, fmt=f_w, col_fmt=b_w)
            dx = MX.gemm(dy_row, w_col, out_dtype=dy.dtype)
        if need_dw:
            mg = getattr(weight, "main_grad", None)
            if mg is not None:
                MX.gemm(dy_col, saved, out=mg, accumulate=True)
            else:
                dw = MX.gemm(dy_col, saved, out_dtype=weight.dtype if weight.dtype != torch.float32 else torch.float32)
        return dx, dw
    if precision == "fp4" and fp4_eligible(M, N, Kd):
        return fp4_backward(dy, saved, weight, need_dx=need_dx, need_dw=need_dw)
    if precision == "fp8" and low_precision(precision, M, N, Kd):
        if need_dw and not isinstance(saved, F8.FP8Operand):
            st = _site(weight, "x", "e4m3")
            st.prepare(saved, _WEIGHT_EPOCH)
            _, saved = F8.quantize(saved, st, want_row=False, want_col=True)
        st = _site(weight, "dy", "e5m2")                 # gradients: e5m2 (range over precision)
        st.prepare(dy, _WEIGHT_EPOCH)
        dy_row, dy_col = F8.quantize(dy, st, want_row=need_dx, want_col=need_dw)
        if need_dx:
            _, w_col = fp8_weight_operands(weight, need_col=True)
            dx = F8.gemm(dy_row, w_col, out_dtype=dy.dtype)
        if need_dw:
            mg = getattr(weight, "main_grad", None)
            if mg is not None:
                F8.gemm(dy_col, saved, out=mg, accumulate=True)
            else:
                dw = F8.gemm(dy_col, saved, out_dtype=weight.dtype if weight.dtype != torch.float32 else torch.float32)
        return dx, dw
    if isinstance(saved, F8.FP8Operand):
        # the forward ran in fp8 but this backward cannot (a dimension of 128): dequantise the saved copy
        saved = F8.dequantize(saved).t().contiguous().to(dy.dtype)
    if need_dx:
        dx = K.gemm(dy, weight, b_mn_major=True)
    if need_dw:
        mg = getattr(weight, "main_grad", None)
        if mg is not None:
            K.gemm(dy, saved, a_mn_major=True, b_mn_major=True, out=mg, accumulate=True)
        else:
            dw = K.gemm(dy, saved, a_mn_major=True, b_mn_major=True, out_dtype=weight.dtype)
    return dx, dw
