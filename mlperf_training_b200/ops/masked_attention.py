"""Attention with document, prefix and window masks, capped scores and a distance bias: raw operators (``functional.masked_attention`` has
their gradients).

The masks of a step are made once, by ``attention_mask``, and shared by its layers: they are intervals of keys for each query (and of queries
for each key), with the tables by which the kernels skip what is not visible (``csrc/attn_mask.cuh``).  The packed samples of the reference's
fine-tuning run carry the boundaries that such a mask is made from (``seq_start_id``, llama2_sft/primus/scripts/convert_dataset.py)."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import call, ptr, stream_ptr, use_kernels

HEAD_DIMS = (64, 128)
SOFTCAPS = (1e-12, 1e18)        # whose squares fp32 holds


@dataclass
class AttentionMask:
    """What each of the last ``Sq`` of ``Skv`` positions sees, for ``B`` sequences; made by ``attention_mask``."""
    B: int
    Sq: int
    Skv: int
    device: torch.device
    buf: torch.Tensor | None = None           # the kernels' tables (CUDA)
    lo: torch.Tensor | None = None            # [B, Sq]: keys [lo, hi) (CPU)
    hi: torch.Tensor | None = None

    def visible(self) -> torch.Tensor:
        """``[B, Sq, Skv]`` truth values."""
        if self.lo is None:
            Sp = -(-self.Sq // 256) * 256
            at = (self.B * (Sp // 128) + self.B * -(-self.Skv // 128)) * 4
            iv = self.buf[at:at + self.B * Sp * 2].view(self.B, Sp, 2)[:, :self.Sq]
            lo, hi = iv[..., 0], iv[..., 1]
        else:
            lo, hi = self.lo, self.hi
        k = torch.arange(self.Skv, device=self.device)
        return (k >= lo[..., None]) & (k < hi[..., None])


def _intervals(B, Sq, Skv, causal, window, documents, prefix):
    at = torch.arange(Skv).expand(B, Skv)
    ids = documents if documents is not None else torch.zeros(B, Skv, dtype=torch.int32)
    start = torch.ones(B, Skv, dtype=torch.bool)
    start[:, 1:] = ids[:, 1:] != ids[:, :-1]
    ds = torch.cummax(torch.where(start, at, 0), 1)[0]
    last = torch.ones_like(start)
    last[:, :-1] = start[:, 1:]

    def next_of(here, value):
        return torch.cummin(torch.where(here, value, Skv).flip(1), 1)[0].flip(1)

    de = next_of(last, at + 1)
    lo = torch.maximum(ds, at - window + 1) if window > 0 else ds
    hi = de
    if causal:
        hi = at + 1
        if prefix is not None:
            bare = next_of(~prefix, at)
            hi = torch.maximum(hi, torch.minimum(bare.gather(1, ds), de))
    pad = ids < 0
    return (torch.where(pad, at, lo)[:, Skv - Sq:].contiguous(), torch.where(pad, at, hi)[:, Skv - Sq:].contiguous())


def attention_mask(B: int, Sq: int, Skv: int | None = None, *, causal: bool = True, window: int = 0, documents: torch.Tensor | None = None,
                   prefix: torch.Tensor | None = None, device=None) -> AttentionMask:
    """The mask of ``B`` sequences whose queries are the last ``Sq`` of ``Skv`` positions (``Sq`` where it is None).

    A query sees keys of its own document: ``documents [B, Skv]`` (int32 or int64) holds an id for each position, a document is a run of equal ids, and
    a position with a negative id is padding, which sees nothing and is not seen.  With ``causal`` it sees keys up to its own position, and
    those of its document's prefix: the leading positions of the document that ``prefix [B, Skv]`` (bool) flags.  With a ``window`` it sees only keys
    less than that many positions behind it."""
    Skv = Sq if Skv is None else Skv
    given = [t for t in (documents, prefix) if t is not None]
    dev = torch.device(device) if device is not None else (given[0].device if given else torch.device("cpu"))
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    if dev.type == "cuda" and _lib.host is not None:
        _lib.require()
        buf = _lib.host.attention_mask(documents, prefix, B, Sq, Skv, int(causal), window, dev.index)
        if buf is not None:
            return AttentionMask(B, Sq, Skv, dev, buf=buf)
    if not 1 <= B <= 2 ** 30 or Sq < 1 or Skv < Sq or Skv > 2 ** 30:
        raise ValueError(f"attention_mask: {B} sequences, {Sq} queries at the end of {Skv} positions (at least one of each)")
    if not 0 <= window < 2 ** 30:
        raise ValueError(f"attention_mask: window {window}")
    if prefix is not None and not causal:
        raise ValueError("attention_mask: a prefix is what a causal mask leaves visible")
    if documents is not None and (documents.shape != (B, Skv) or documents.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"attention_mask: documents [{B}, {Skv}] in int32 or int64, not {list(documents.shape)} in {documents.dtype}")
    if prefix is not None and (prefix.shape != (B, Skv) or prefix.dtype != torch.bool):
        raise ValueError(f"attention_mask: prefix [{B}, {Skv}] of truth values, not {list(prefix.shape)} in {prefix.dtype}")
    if any(t.device != dev for t in given):
        raise ValueError(f"attention_mask: documents and prefix on {dev}")
    if dev.type != "cuda":
        lo, hi = _intervals(B, Sq, Skv, causal, window, documents, prefix)
        return AttentionMask(B, Sq, Skv, dev, lo=lo, hi=hi)
    n = int(_lib.load().b200_attn_mask_ints(B, Sq, Skv))
    buf = torch.empty(n, dtype=torch.int32, device=dev)
    documents = None if documents is None else documents.contiguous()
    prefix = None if prefix is None else prefix.contiguous()
    with _lib.on_device_of(buf):
        call("b200_attn_mask", ptr(documents), int(documents is not None and documents.dtype == torch.int64), ptr(prefix), B, Sq, Skv, int(causal),
             int(window), ptr(buf), stream_ptr())
    return AttentionMask(B, Sq, Skv, dev, buf=buf)


def _check(q, k, v, mask, scale, softcap, slopes, sink) -> None:
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"masked_attention: q [B, Sq, Hq, D] and k, v [B, Skv, Hkv, D], not {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    B, Sq, Hq, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    if (mask.B, mask.Sq, mask.Skv) != (B, Sq, Skv) or mask.device != q.device:
        raise ValueError(f"masked_attention: a mask of {mask.B} x {mask.Sq} x {mask.Skv} on {mask.device} for {B} x {Sq} x {Skv} on {q.device}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"masked_attention: {Hq} query heads over {Hkv} key heads")
    if not (q.dtype == k.dtype == v.dtype) or any(t.device != q.device for t in (k, v)):
        raise ValueError(f"masked_attention: q, k, v of one type on one device, not {q.dtype}, {k.dtype}, {v.dtype} on {q.device}, {k.device}, {v.device}")
    if q.is_cuda and (q.dtype != torch.bfloat16 or D not in HEAD_DIMS):
        raise ValueError(f"masked_attention: bf16 with head dim 64 or 128, not {q.dtype} with {D}")
    if not (0.0 < scale < math.inf and (softcap == 0.0 or SOFTCAPS[0] <= softcap <= SOFTCAPS[1])):
        raise ValueError(f"masked_attention: scale {scale} (above 0), softcap {softcap} (0: none, else {SOFTCAPS[0]} to {SOFTCAPS[1]})")
    for name, t in (("slopes", slopes), ("sink", sink)):
        if t is not None and (t.shape != (Hq,) or t.device != q.device or not t.is_floating_point()):
            raise ValueError(f"masked_attention: {name} [{Hq}] on {q.device}, not {list(t.shape)} in {t.dtype} on {t.device}")


def constant_slopes(slopes) -> None:
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("masked_attention: the slopes of the distance bias are constants (no gradient goes to them)")


def _bshd(t: torch.Tensor):
    """``t [B, S, H, D]`` as the kernels read it, with its row and batch pitch: heads contiguous in a row, 16-byte aligned rows, no overlap."""
    B, S, H, D = t.shape
    w = H * D
    row = t.stride(1) if S > 1 else w
    batch = t.stride(0) if B > 1 else S * row
    if ((t.stride(3) != 1 and D > 1) or (t.stride(2) != D and H > 1) or row < w or batch < w or row % 8 or batch % 8 or t.data_ptr() % 16):
        t = t.contiguous()
        row, batch = w, S * w
        if t.data_ptr() % 16:
            t = t.clone()
    return t, row, batch


def _scores(q, k, mask, scale, softcap, slopes):
    """Scores ``[B, Hq, Sq, Skv]`` with -inf where nothing is visible (CPU)."""
    group, Sq, Skv = q.shape[2] // k.shape[2], mask.Sq, mask.Skv
    s = torch.matmul(q.permute(0, 2, 1, 3), k.permute(0, 2, 3, 1).repeat_interleave(group, 1)) * scale
    if softcap > 0:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        at = torch.arange(Skv, dtype=s.dtype)
        s = s - slopes.to(s.dtype)[:, None, None] * (at[Skv - Sq:, None] - at).abs()
    return s.masked_fill(~mask.visible()[:, None], -math.inf)


def _reference(q, k, v, mask, scale, softcap, slopes, sink):
    """``(out, lse)``; rows that see nothing give 0 (and no NaN to their gradients)."""
    s = _scores(q, k, mask, scale, softcap, slopes)
    if sink is not None:
        s = torch.cat([s, sink.to(s.dtype).view(1, -1, 1, 1).expand(*s.shape[:3], 1)], -1)
    none = (s == -math.inf).all(-1, keepdim=True)
    lse = torch.logsumexp(torch.where(none, 0.0, s), -1)
    p = torch.where(none, 0.0, torch.exp(s - lse[..., None]))[..., :mask.Skv]
    seen = mask.visible().any(1)[:, :, None, None]                       # (0 times what lies in padding is 0)
    vv = torch.where(seen, v, 0.0).permute(0, 2, 1, 3).repeat_interleave(q.shape[2] // k.shape[2], 1)
    return torch.matmul(p, vv).permute(0, 2, 1, 3), torch.where(none[..., 0], -math.inf, lse)


def masked_attention_fwd(q, k, v, mask: AttentionMask, *, scale: float | None = None, softcap: float = 0.0, slopes: torch.Tensor | None = None,
                         sink: torch.Tensor | None = None, for_backward: bool = False):
    """``(out [B, Sq, Hq, D], lse fp32 [B, Hq, Sq], low)``; ``low`` (with ``for_backward``, on the GPU) is what ``out`` has lost to bf16."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    _check(q, k, v, mask, scale, softcap, slopes, sink)
    B, Sq, Hq, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    if not use_kernels(q):
        o, lse = _reference(*(t.detach().double() for t in (q, k, v)), mask, scale, softcap, slopes, sink)
        return o.to(q.dtype).contiguous(), lse.float(), None
    (q, q_row, q_batch), (k, k_row, k_batch), (v, v_row, v_batch) = _bshd(q), _bshd(k), _bshd(v)
    out = torch.empty((B, Sq, Hq, D), dtype=q.dtype, device=q.device)
    low = torch.empty_like(out) if for_backward else None
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device)
    slopes = None if slopes is None else slopes.detach().float().contiguous()
    sink = None if sink is None else sink.detach().float().contiguous()
    lib = _lib.load()
    with _lib.on_device_of(q):
        if not for_backward and lib.b200_attn_masked_few_rows(B, Sq, Hq, Hkv):
            n = int(lib.b200_attn_masked_rows_workspace(B, Sq, Skv, Hq, Hkv, D))
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
            call("b200_attn_masked_rows", ptr(q), ptr(k), ptr(v), ptr(out), ptr(lse), ptr(sink), ptr(slopes), ptr(mask.buf), B, Sq, Skv, Hq, Hkv,
                 D, q_row, k_row, v_row, q_batch, k_batch, v_batch, float(scale), float(softcap), ptr(ws), n, stream_ptr())
            return out, lse, None
        n = int(lib.b200_attn_masked_fwd_workspace(B, Sq, Skv, Hq, D))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        call("b200_attn_masked_fwd", ptr(q), ptr(k), ptr(v), ptr(out), ptr(low), ptr(lse), ptr(sink), ptr(slopes), ptr(mask.buf), B, Sq, Skv, Hq,
             Hkv, D, q_row, k_row, v_row, q_batch, k_batch, v_batch, float(scale), float(softcap), ptr(ws), n, stream_ptr())
    return out, lse, low


def masked_attention_bwd(dout, q, k, v, out, low, lse, mask: AttentionMask, *, scale: float | None = None, softcap: float = 0.0,
                         slopes: torch.Tensor | None = None, sink: torch.Tensor | None = None, dk_out=None, dv_out=None):
    """``(dq fp32 [B, Sq, Hq, D], dk, dv, dsink or None)``; ``dk_out`` / ``dv_out`` may be views into a packed gradient buffer."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    _check(q, k, v, mask, scale, softcap, slopes, sink)
    B, Sq, Hq, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    if dout.shape != q.shape or dout.device != q.device:
        raise ValueError(f"masked_attention: gradient {list(q.shape)} on {q.device}, not {list(dout.shape)} on {dout.device}")
    if not use_kernels(q):
        ins = [t.detach().double().requires_grad_(True) for t in (q, k, v) + (() if sink is None else (sink,))]
        with torch.enable_grad():
            o, _ = _reference(*ins[:3], mask, scale, softcap, slopes, ins[3] if sink is not None else None)
        g = torch.autograd.grad(o, ins, dout.double())
        dk, dv = g[1].to(k.dtype), g[2].to(v.dtype)
        dk = dk if dk_out is None else dk_out.copy_(dk)
        dv = dv if dv_out is None else dv_out.copy_(dv)
        return g[0].float(), dk, dv, (g[3].float() if sink is not None else None)
    (q, q_row, q_batch), (k, k_row, k_batch), (v, v_row, v_batch) = _bshd(q), _bshd(k), _bshd(v)
    dout = dout.to(q.dtype).contiguous()
    dout = dout if dout.data_ptr() % 16 == 0 else dout.clone()
    dq = torch.empty((B, Sq, Hq, D), dtype=torch.float32, device=q.device)
    dk = dk_out if dk_out is not None else torch.empty((B, Skv, Hkv, D), dtype=k.dtype, device=k.device)
    dv = dv_out if dv_out is not None else torch.empty((B, Skv, Hkv, D), dtype=v.dtype, device=v.device)
    (wk, dk_row, dk_batch), (wv, dv_row, dv_batch) = _bshd(dk), _bshd(dv)
    delta = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device)
    n = int(_lib.load().b200_attn_masked_bwd_workspace(B, Sq, Skv, Hq, Hkv, D))
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    slopes = None if slopes is None else slopes.detach().float().contiguous()
    with _lib.on_device_of(q):
        call("b200_attn_masked_bwd", ptr(q), ptr(k), ptr(v), ptr(out), ptr(low), ptr(dout), ptr(lse), ptr(delta), ptr(dq), ptr(wk), ptr(wv),
             ptr(slopes), ptr(mask.buf), B, Sq, Skv, Hq, Hkv, D, q_row, k_row, v_row, dk_row, dv_row, q_batch, k_batch, v_batch, dk_batch, dv_batch,
             float(scale), float(softcap), ptr(ws), n, stream_ptr())
    if wk is not dk:
        dk.copy_(wk)
    if wv is not dv:
        dv.copy_(wv)
    dsink = None
    if sink is not None:
        # of the extra column, which carries no value: -sum over rows of its probability times delta (0 where the row has neither a key nor a sink)
        at = sink.detach().float().view(1, Hq, 1)
        dsink = -(torch.where(at == -math.inf, 0.0, torch.exp(at - lse)) * delta).sum(dim=(0, 2))
    return dq, dk, dv, dsink
