"""Operators of low-precision training, one pass each, on one GPU: the RMS norm with a micro-scaled output, MXFP4
quantisation, the MXFP4 product and linear layer, and the gated feed-forward block.

A case is a dict of plain values; ``kind`` says which operator it takes:

    norm    addition of a residual, RMS norm, MXFP8 copies of the result (along the rows, optionally along the columns
            too), optionally the backward pass
    quant   MXFP4 copies of a matrix, rounded to nearest or stochastically from given bytes, optionally with the
            16-row Hadamard transform ahead of the column-wise copy
    gemm    a linear layer with a frozen 4-bit weight: the activations quantised to MXFP4, the product
    linear  an MXFP4 linear layer in training: output, gradient of the input and of the weight
    gated   gated feed-forward block (gate, up, SiLU, down projection), forward alone or with its backward pass

``listed()`` are fixed sizes, ``draw(rng)`` gives others of the same ranges.  Quantised results are returned as the
values they stand for (bf16 holds every one of them).
"""
import math

import torch

own = False

EPS = 1e-5
DEV = "cuda"
BF16 = torch.bfloat16


# --------------------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------------------
def listed():
    return [
        # generation: one token's activations on the way into a block-scaled linear
        dict(name="norm_token", kind="norm", T=1, D=4096, residual=True, cols=False, train=False),
        # evaluation of a mixture-of-experts decoder (width 2880) on a ragged batch
        dict(name="norm_ragged", kind="norm", T=1337, D=2880, residual=False, cols=False, train=False),
        # training of an 8B decoder: two sequences of 8192, both copies and the backward pass
        dict(name="norm_train", kind="norm", T=16384, D=4096, residual=True, cols=True, train=True),
        # a handful of activation rows, where a launch is most of the time
        dict(name="quant_rows", kind="quant", R=16, C=4096, rows=True, cols=False, noise=False, hadamard=False),
        # an up-projection's weight after an optimizer step: both copies, rounded to nearest
        dict(name="quant_weight", kind="quant", R=14336, C=4096, rows=True, cols=True, noise=False, hadamard=False),
        # an output gradient of an odd number of tokens: both copies, stochastic rounding, Hadamard transform
        dict(name="quant_grad", kind="quant", R=4011, C=14336, rows=True, cols=True, noise=True, hadamard=True),
        # one token through a gate | up projection whose weight is kept in 4 bits
        dict(name="gemm_token", kind="gemm", M=1, N=28672, K=4096, bias=False, residual=False),
        # ragged rows, a contraction that ends inside a tile, bias and residual
        dict(name="gemm_ragged", kind="gemm", M=2003, N=5120, K=2880, bias=True, residual=True),
        # evaluation: two sequences of 8192 through the gate | up projection of an 8B decoder
        dict(name="gemm_large", kind="gemm", M=16384, N=28672, K=4096, bias=False, residual=False),
        # a down projection in training: forward and both gradients
        dict(name="linear_train", kind="linear", M=8192, N=4096, K=14336),
        # generation: a few tokens through the feed-forward block
        dict(name="gated_eval", kind="gated", T=7, D=4096, F=14336, residual=True, train=False),
        # training of the block on half a sequence
        dict(name="gated_train", kind="gated", T=4096, D=4096, F=14336, residual=True, train=True),
    ]


def _log(rng, lo, hi, step=1):
    """An integer between lo and hi, spread over its logarithm, rounded to a multiple of ``step``."""
    v = int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    v = min(hi, max(lo, v)) // step * step
    v = max(step, v)
    return v + step if v == 3072 else v


def draw(rng):
    kind = rng.choice(["norm", "quant", "gemm", "linear", "gated"])
    flag = lambda: rng.random() < 0.5
    if kind == "norm":
        D = _log(rng, 128, 8192, 32)
        return dict(kind=kind, T=_log(rng, 1, 16384 * 4096 // D), D=D, residual=flag(), cols=flag(), train=flag())
    if kind == "quant":
        C = _log(rng, 64, 14336, 32)
        rows = flag()
        return dict(kind=kind, R=_log(rng, 1, min(32768, 14336 * 4096 // C)), C=C, rows=rows, cols=flag() or not rows, noise=flag(),
                    hadamard=flag())
    if kind == "gemm":
        N, K = _log(rng, 64, 28672, 8), _log(rng, 64, 14336, 32)
        return dict(kind=kind, M=_log(rng, 1, min(16384, 16384 * 28672 * 4096 // (N * K))), N=N, K=K, bias=flag(), residual=flag())
    if kind == "linear":
        N, K = _log(rng, 128, 14336, 32), _log(rng, 128, 14336, 32)
        return dict(kind=kind, M=_log(rng, 1, min(16384, 8192 * 4096 * 14336 // (N * K))), N=N, K=K)
    D, F = _log(rng, 256, 4096, 8), _log(rng, 256, 14336, 8)
    return dict(kind=kind, T=_log(rng, 1, 4096), D=D, F=F, residual=flag(), train=flag())


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _acts(g, rows, cols, std=1.0):
    """Activations: normal, with a few columns ten times as large (the outlier channels of a decoder)."""
    x = torch.randn(rows, cols, generator=g, device=DEV) * std
    x *= 1 + 9 * (torch.rand(cols, generator=g, device=DEV) < 1 / 256)
    return x.to(BF16)


def prepare(case, seed):
    g, k = _gen(seed), case["kind"]
    s = dict(case)
    if k == "norm":
        T, D = case["T"], case["D"]
        s["x"] = _acts(g, T, D)
        s["res"] = _acts(g, T, D, 3.0) if case["residual"] else None
        s["w"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(BF16)
        if case["train"]:
            s["dy"], s["dh"] = _acts(g, T, D, 1e-3), _acts(g, T, D, 1e-3)
    elif k == "quant":
        R, C = case["R"], case["C"]
        # gradients span many powers of two from row to row
        scale = torch.exp2(torch.randint(-12, 1, (R, 1), generator=g, device=DEV).float())
        s["x"] = (torch.randn(R, C, generator=g, device=DEV) * scale).to(BF16)
        s["u"] = torch.randint(0, 256, (R, C), generator=g, device=DEV, dtype=torch.uint8) if case["noise"] else None
    elif k == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _acts(g, M, K)
        # a weight that is kept in 4 bits, as the values it stands for
        s["weight"] = _mx_rows(torch.randn(N, K, generator=g, device=DEV) * 0.02, "e2m1").to(BF16)
        s["b"] = torch.randn(N, generator=g, device=DEV).to(BF16) if case["bias"] else None
        s["r"] = _acts(g, M, N) if case["residual"] else None
    elif k == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = _acts(g, M, K).requires_grad_(True)
        s["weight"] = (torch.randn(N, K, generator=g, device=DEV) * 0.02).to(BF16).requires_grad_(True)
        s["dy"] = _acts(g, M, N, 1e-3)
        s["u"] = torch.randint(0, 256, (M, N), generator=g, device=DEV, dtype=torch.uint8)
    else:
        T, D, F, t = case["T"], case["D"], case["F"], case["train"]
        s["x"] = _acts(g, T, D).requires_grad_(t)
        s["w_gu"] = (torch.randn(2 * F, D, generator=g, device=DEV) * 0.02).to(BF16).requires_grad_(t)
        s["w_down"] = (torch.randn(D, F, generator=g, device=DEV) * 0.02).to(BF16).requires_grad_(t)
        s["r"] = _acts(g, T, D).requires_grad_(t) if case["residual"] else None
        s["dy"] = _acts(g, T, D, 1e-3) if t else None
    return s


# --------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# --------------------------------------------------------------------------------------
FORMATS = {"e4m3": (3, -6, 448.0), "e2m1": (1, 0, 6.0)}      # mantissa bits, smallest exponent, largest value


def _mx_rows(v, fmt, u=None):
    """The values that blocks of 32 along the rows of ``v`` have in ``fmt`` with one power-of-two scale each."""
    bits, e_min, top = FORMATS[fmt]
    b = v.reshape(v.shape[0], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True) / top)
    e = torch.where(m == 0.5, e - 1, e).clamp(-127, 127)
    y = torch.ldexp(b, -e)
    quantum = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=e_min).float() - bits)
    t = y.abs() / quantum
    t = torch.round(t) if u is None else torch.floor(t + (u.reshape(b.shape).float() + 0.5) / 256)
    return torch.ldexp(torch.copysign((t * quantum).clamp(max=top), y), e).reshape(v.shape)


def _pad_rows(v, to, value=0):
    return torch.nn.functional.pad(v, (0, 0, 0, -v.shape[0] % to), value=value)


def _hadamard(v):
    """Groups of 16 rows times the orthonormal Hadamard matrix of that size: H[i, j] = (-1)^popcount(i & j) / 4."""
    i = torch.arange(16, device=v.device)
    both = i[:, None] & i[None, :]
    ones = (both & 1) + (both >> 1 & 1) + (both >> 2 & 1) + (both >> 3)
    h = (1 - 2 * (ones % 2)).to(v.dtype) / 4
    return torch.matmul(h, v.reshape(-1, 16, v.shape[1])).reshape(v.shape)


def _mx_cols(v, fmt, hadamard=False, u=None, to=32):
    """The column-wise copy, transposed: rows are filled up with zeros (and their bytes with 128) to a multiple of ``to``."""
    v = _pad_rows(v, to)
    v = _hadamard(v) if hadamard else v
    return _mx_rows(v.t().contiguous(), fmt, None if u is None else _pad_rows(u, to, 128).t().contiguous())


def _plain(s):
    k = s["kind"]
    if k == "norm":
        h = s["x"].float() if s["res"] is None else (s["x"].float() + s["res"].float()).to(BF16).float()
        rstd = torch.rsqrt((h * h).mean(-1) + EPS)
        xn = h * rstd[:, None]
        n = xn * s["w"].float()
        out = {"rows": _mx_rows(n, "e4m3").to(BF16), "rstd": rstd}
        if s["res"] is not None:
            out["h"] = h.to(BF16)
        if s["cols"]:
            out["cols"] = _mx_cols(n, "e4m3", to=128).to(BF16)
        if s["train"]:
            dy = s["dy"].float()
            gr = dy * s["w"].float()
            out["dx"] = (rstd[:, None] * (gr - xn * (gr * xn).mean(-1, keepdim=True)) + s["dh"].float()).to(BF16)
            out["dw"] = (dy * xn).sum(0)
        return out
    if k == "quant":
        x, out = s["x"].float(), {}
        if s["rows"]:
            out["rows"] = _mx_rows(x, "e2m1", s["u"]).to(BF16)
        if s["cols"]:
            out["cols"] = _mx_cols(x, "e2m1", s["hadamard"], s["u"]).to(BF16)
        return out
    if k == "gemm":
        y = _mx_rows(s["x"].float(), "e2m1") @ s["weight"].float().t()
        y = y if s["b"] is None else y + s["b"].float()
        return (y if s["r"] is None else y + s["r"].float()).to(BF16)
    with torch.no_grad():
        if k == "linear":
            x, w, dy = s["x"].float(), s["weight"].float(), s["dy"].float()
            y = _mx_rows(x, "e2m1") @ _mx_rows(w, "e2m1").t()
            dx = _mx_rows(dy, "e2m1", s["u"]) @ _mx_cols(w, "e2m1").t()
            dw = _mx_cols(dy, "e2m1", True, s["u"]) @ _mx_cols(x, "e2m1", True).t()
            return {"y": y.to(BF16), "dx": dx.to(BF16), "dw": dw.to(BF16)}
        x, wd, F = s["x"].float(), s["w_down"].float(), s["F"]
        wg, wu = s["w_gu"][:F].float(), s["w_gu"][F:].float()
        gate, up = x @ wg.t(), x @ wu.t()
        sg = torch.sigmoid(gate)
        a = gate * sg * up
        y = a @ wd.t()
        y = y if s["r"] is None else y + s["r"].float()
        if not s["train"]:
            return y.to(BF16)
        dy = s["dy"].float()
        da = dy @ wd
        dg, du = da * up * sg * (1 + gate * (1 - sg)), da * gate * sg
        out = {"y": y, "dx": dg @ wg + du @ wu, "dw_gu": torch.cat([dg.t() @ x, du.t() @ x]), "dw_down": dy.t() @ a}
        if s["r"] is not None:
            out["dr"] = dy
        return {n: v.to(BF16) for n, v in out.items()}


# --------------------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------------------
def _own(s):
    from mlperf_training_b200.ops import functional as F
    from mlperf_training_b200.ops import kernels as K
    from mlperf_training_b200.ops import linear as L
    from mlperf_training_b200.ops import mxfp4, mxfp8
    from mlperf_training_b200.ops.norm_mx import rms_norm_quantize
    k = s["kind"]
    if k == "norm":
        row, col, h, rstd = rms_norm_quantize(s["x"], s["w"], EPS, residual=s["res"], row_tile=mxfp8.A_TILE,
                                              col_tile=mxfp8.b_tile(s["D"]) if s["cols"] else None)
        out = {"rows": mxfp4.dequantize(row, BF16), "rstd": rstd}
        if s["res"] is not None:
            out["h"] = h
        if s["cols"]:
            out["cols"] = mxfp4.dequantize(col, BF16)
        if s["train"]:
            out["dx"], out["dw"], _ = K.norm_bwd(s["dy"], h, s["w"], None, None, rstd, dres=s["dh"])
        return out
    if k == "quant":
        row, col = mxfp4.quantize(s["x"], row_tile=mxfp4.A_TILE if s["rows"] else None,
                                  col_tile=mxfp4.b_tile(s["C"]) if s["cols"] else None, noise=s["u"], hadamard=s["hadamard"])
        out = {}
        if s["rows"]:
            out["rows"] = mxfp4.dequantize(row, BF16)
        if s["cols"]:
            out["cols"] = mxfp4.dequantize(col, BF16)
        return out
    if k == "gemm":
        with torch.no_grad():
            return F.mxfp4_linear(s["x"], s["weight"], bias=s["b"], residual=s["r"])
    if k == "linear":
        L.bump_weight_epoch()                   # the weight has changed since the last step: its 4-bit copies are made anew
        y = F.mxfp4_linear(s["x"], s["weight"], noise=s["u"])
        dx, dw = torch.autograd.grad(y, [s["x"], s["weight"]], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if not s["train"]:
        with torch.no_grad():
            return F.gated_mlp(s["x"], s["w_gu"], s["w_down"], residual=s["r"])
    y = F.gated_mlp(s["x"], s["w_gu"], s["w_down"], residual=s["r"])
    over = [s["x"], s["w_gu"], s["w_down"]] + ([s["r"]] if s["r"] is not None else [])
    grads = torch.autograd.grad(y, over, s["dy"])
    return {"y": y.detach(), **dict(zip(["dx", "dw_gu", "dw_down", "dr"], grads))}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------
def work(case):
    k = case["kind"]
    if k == "norm":
        T, D = case["T"], case["D"]
        b = 2 * T * D + 2 * T * D + 4 * T + 2 * D                       # x, row copy, rstd, weight
        b += 4 * T * D if case["residual"] else 0                       # residual, sum
        b += 2 * D * (-(-T // 128) * 128) if case["cols"] else 0
        b += 6 * T * D + 4 * D if case["train"] else 0                  # dy, dh, dx, dw
        return {"bytes": b, "flops": T * D * (8 + 10 * case["train"])}
    if k == "quant":
        R, C = case["R"], case["C"]
        b = 2 * R * C + (R * C if case["noise"] else 0)
        b += 2 * R * C if case["rows"] else 0
        b += 2 * C * (-(-R // 32) * 32) if case["cols"] else 0
        return {"bytes": b, "flops": R * C * (4 * case["rows"] + (4 + 4 * case["hadamard"]) * case["cols"])}
    if k == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        b = 2 * M * K + N * K // 2 + N * K // 32 + 2 * M * N
        b += (2 * N if case["bias"] else 0) + (2 * M * N if case["residual"] else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    if k == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (2 * M * K + 2 * N * K + 2 * M * N) + M * N, "flops": 6 * M * N * K}
    T, D, F = case["T"], case["D"], case["F"]
    b = 2 * (3 * D * F + 2 * T * D) + (2 * T * D if case["residual"] else 0)
    if case["train"]:
        b += 2 * (3 * D * F + 2 * T * D) + (2 * T * D if case["residual"] else 0)
    return {"bytes": b, "flops": 6 * T * D * F * (3 if case["train"] else 1)}


# --------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------
def _exact_e8m0(amax, top):
    """The smallest power of two that is not below amax / top (2^-127 for zero)."""
    p = torch.exp2(torch.ceil(torch.log2(amax / top)))
    p = torch.where(p / 2 * top >= amax, p / 2, p)            # the logarithm may round across a power of two
    p = torch.where(p * top < amax, p * 2, p)
    return torch.where(amax > 0, p, torch.full_like(p, 2.0 ** -127))


def _exact_grid(fmt):
    if fmt == "e2m1":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    return torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()


def _exact_mx(v, fmt, u=None):
    grid = _exact_grid(fmt)
    b = v.reshape(v.shape[0], -1, 32)
    p = _exact_e8m0(b.abs().amax(-1, keepdim=True), float(grid[-1]))
    a = (b / p).abs()
    lo = (torch.searchsorted(grid, a.reshape(-1), right=True) - 1).clamp(max=len(grid) - 2).reshape(a.shape)
    part = (a - grid[lo]) / (grid[lo + 1] - grid[lo])         # place between the neighbours
    if u is None:
        up = (part > 0.5) | ((part == 0.5) & (lo % 2 == 1))   # codes alternate between even and odd
    else:
        up = part + (u.reshape(b.shape).double() + 0.5) / 256 >= 1
    return (torch.sign(b) * grid[lo + up] * p).reshape(v.shape)


def _exact_hadamard(v):
    """The transform as four steps of sums and differences."""
    x = v.reshape(-1, 2, 2, 2, 2, v.shape[1])
    x = torch.stack([x.select(1, 0) + x.select(1, 1), x.select(1, 0) - x.select(1, 1)], 1)
    x = torch.stack([x.select(2, 0) + x.select(2, 1), x.select(2, 0) - x.select(2, 1)], 2)
    x = torch.stack([x.select(3, 0) + x.select(3, 1), x.select(3, 0) - x.select(3, 1)], 3)
    x = torch.stack([x.select(4, 0) + x.select(4, 1), x.select(4, 0) - x.select(4, 1)], 4)
    return x.reshape(v.shape) / 4


def _exact_cols(v, fmt, hadamard=False, u=None, to=32):
    n = -v.shape[0] % to
    v = torch.cat([v, v.new_zeros(n, v.shape[1])])
    if u is not None:
        u = torch.cat([u, u.new_full((n, u.shape[1]), 128)]).t().contiguous()
    return _exact_mx((_exact_hadamard(v) if hadamard else v).t().contiguous(), fmt, u)


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    d = lambda n: s[n].double()
    k = case["kind"]
    if k == "norm":
        h = d("x") if s["res"] is None else (d("x") + d("res")).to(BF16).double()
        ms = h.square().sum(1) / h.shape[1] + EPS
        n = h / ms.sqrt()[:, None]
        y = n * d("w")
        out = {"rows": _exact_mx(y, "e4m3"), "rstd": 1 / ms.sqrt()}
        if s["res"] is not None:
            out["h"] = h
        if case["cols"]:
            out["cols"] = _exact_cols(y, "e4m3", to=128)
        if case["train"]:
            q = d("dy") * d("w")
            out["dx"] = (q - n * ((q * n).sum(1, keepdim=True) / h.shape[1])) / ms.sqrt()[:, None] + d("dh")
            out["dw"] = (d("dy") * n).sum(0)
        return out
    if k == "quant":
        out = {}
        if case["rows"]:
            out["rows"] = _exact_mx(d("x"), "e2m1", s["u"])
        if case["cols"]:
            out["cols"] = _exact_cols(d("x"), "e2m1", case["hadamard"], s["u"])
        return out
    if k == "gemm":
        y = torch.matmul(_exact_mx(d("x"), "e2m1"), d("weight").t())
        y = y + d("b") if s["b"] is not None else y
        return y + d("r") if s["r"] is not None else y
    if k == "linear":
        return {"y": torch.matmul(_exact_mx(d("x"), "e2m1"), _exact_mx(d("weight"), "e2m1").t()),
                "dx": torch.matmul(_exact_mx(d("dy"), "e2m1", s["u"]), _exact_cols(d("weight"), "e2m1").t()),
                "dw": torch.matmul(_exact_cols(d("dy"), "e2m1", True, s["u"]), _exact_cols(d("x"), "e2m1", True).t())}
    F = case["F"]
    gu = torch.matmul(d("x"), d("w_gu").t())
    gate, up = gu[:, :F], gu[:, F:]
    act = gate / (1 + torch.exp(-gate))
    y = torch.matmul(act * up, d("w_down").t()) + (d("r") if s["r"] is not None else 0)
    if not case["train"]:
        return y
    da = torch.matmul(d("dy"), d("w_down"))
    slope = (1 + torch.exp(-gate) + gate * torch.exp(-gate)) / (1 + torch.exp(-gate)).square()
    dgu = torch.cat([da * up * slope, da * act], 1)
    out = {"y": y, "dx": torch.matmul(dgu, d("w_gu")), "dw_gu": torch.matmul(dgu.t(), d("x")),
           "dw_down": torch.matmul(d("dy").t(), act * up)}
    if s["r"] is not None:
        out["dr"] = d("dy")
    return out
