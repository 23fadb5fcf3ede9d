"""Masked attention on the CPU: masks against a walk from query to key, output and gradients against the definition, refusals."""
import pytest
import torch

from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import masked_attention as MA
from tests import masked_oracle as O


def documents(B, S, kind, seed=0):
    """Ids [B, S]: "one", "few" documents, "many" (one to four positions), "padded" at the end, "left" padded, "holes" of padding, "same" ids again
    for another document, "none" live."""
    g = torch.Generator().manual_seed(seed + 17 * S + B)
    if kind == "one":
        return torch.zeros(B, S, dtype=torch.int32)
    p = {"many": 0.4, "few": 4 / S}.get(kind, 5 / S)
    ids = torch.cumsum((torch.rand(B, S, generator=g) < p).int(), 1).int()
    if kind == "padded":
        for b in range(B):
            ids[b, S - (b + 1) * S // (B + 2):] = -1
    if kind == "left":
        for b in range(B):
            ids[b, :b * S // B] = -7 - b
    if kind == "holes":
        ids[torch.rand(B, S, generator=g) < 0.15] = -1
    if kind == "same":
        ids %= 2
    if kind == "none":
        ids[:] = -1
    return ids


def flags(B, S, seed=0):
    return torch.rand(B, S, generator=torch.Generator().manual_seed(seed + S)) < 0.7


MASKS = [dict(), dict(causal=False), dict(window=3), dict(causal=False, window=5), dict(prefix=True), dict(prefix=True, window=4)]
KINDS = ["one", "few", "many", "padded", "left", "holes", "same", "none"]


def make(B, Sq, Skv, kind, m):
    kw = dict(m)
    ids = documents(B, Skv, kind) if kind != "absent" else None
    if kw.get("prefix"):
        kw["prefix"] = flags(B, Skv)
    return dict(documents=ids, **kw)


@pytest.mark.parametrize("m", MASKS, ids=str)
@pytest.mark.parametrize("kind", KINDS + ["absent"])
@pytest.mark.parametrize("B,Sq,Skv", [(1, 1, 1), (2, 9, 9), (3, 40, 40), (2, 1, 30), (2, 5, 33)])
def test_mask_is_its_definition(B, Sq, Skv, kind, m):
    kw = make(B, Sq, Skv, kind, m)
    mask = F.attention_mask(B, Sq, Skv, **kw)
    assert torch.equal(mask.visible(), O.visible(B, Sq, Skv, **kw))
    if kw["documents"] is not None:
        again = F.attention_mask(B, Sq, Skv, **{**kw, "documents": kw["documents"].long()})
        assert torch.equal(again.visible(), mask.visible())


SCORES = [dict(), dict(softcap=2.0), dict(slopes=True), dict(softcap=3.0, slopes=True, sink=True), dict(sink=True), dict(scale=0.5)]


def tensors(B, Sq, Skv, Hq, Hkv, D, score, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed + Sq + Skv)
    q, k, v, do = (torch.randn(B, s, h, D, generator=g).to(dtype) for s, h in ((Sq, Hq), (Skv, Hkv), (Skv, Hkv), (Sq, Hq)))
    kw = dict(score)
    if kw.get("slopes"):
        kw["slopes"] = torch.exp2(-8 * torch.arange(1, Hq + 1).float() / Hq)
    if kw.get("sink"):
        kw["sink"] = torch.randn(Hq, generator=g)
    return q, k, v, do, kw


def oracle(q, k, v, do, ok, kw):
    ins = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    sink = kw["sink"].double().requires_grad_(True) if kw.get("sink") is not None else None
    y = O.attention(*ins, ok, **{**kw, "sink": sink})
    return [y.detach()] + list(torch.autograd.grad(y, ins + ([sink] if sink is not None else []), do.double()))


@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("kind,m", [("few", MASKS[0]), ("holes", MASKS[4]), ("padded", MASKS[3]), ("none", MASKS[0]), ("left", MASKS[2])], ids=str)
@pytest.mark.parametrize("B,Sq,Skv", [(2, 12, 12), (2, 3, 17)])
def test_attention_is_its_definition(B, Sq, Skv, kind, m, score):
    kw = make(B, Sq, Skv, kind, m)
    mask = F.attention_mask(B, Sq, Skv, **kw)
    q, k, v, do, s = tensors(B, Sq, Skv, 4, 2, 8, score)
    want = oracle(q, k, v, do, O.visible(B, Sq, Skv, **kw), s)
    ins = [t.requires_grad_(True) for t in (q, k, v)] + ([s["sink"].requires_grad_(True)] if "sink" in s else [])
    y = F.masked_attention(q, k, v, mask, **s)
    got = [y.detach()] + list(torch.autograd.grad(y, ins, do))
    for a, b in zip(got, want):
        # 64-bit arithmetic on both sides, one rounding to fp32
        assert a.dtype == torch.float32 and torch.allclose(a.double(), b, rtol=2 ** -24 * 1.01, atol=1e-13)
    with torch.no_grad():
        assert torch.equal(F.masked_attention(q, k, v, mask, **s), y)


@pytest.mark.parametrize("score", SCORES[1:4], ids=str)
def test_gradient_against_differences(score):
    kw = make(1, 6, 6, "few", MASKS[4])
    ok = O.visible(1, 6, 6, **kw)
    q, k, v, do, s = tensors(1, 6, 6, 2, 1, 4, score)
    grads = oracle(q, k, v, do, ok, s)[1:4]
    h = 1e-5
    for n, (t, g) in enumerate(zip((q, k, v), grads)):
        for i in range(0, t.numel(), 3):
            side = []
            for e in (h, -h):
                x = [a.detach().double().clone() for a in (q, k, v)]
                x[n].view(-1)[i] += e
                side.append((O.attention(*x, ok, **{**s, "sink": s["sink"].double() if "sink" in s else None}) * do.double()).sum())
            assert abs((side[0] - side[1]) / (2 * h) - g.reshape(-1)[i]) < 1e-8


def test_what_padding_holds_does_not_matter():
    ids = torch.tensor([[0, 0, -1, 1, 1, -1]])
    mask = F.attention_mask(1, 6, documents=ids)
    q, k, v, _, _ = tensors(1, 6, 6, 2, 2, 8, {})
    ref = F.masked_attention(q, k, v, mask)
    for t in (q, k, v):
        t[:, 2] = float("nan")
        t[:, 5] = float("inf")
    assert torch.equal(F.masked_attention(q, k, v, mask), ref)


def test_packed_form_with_rotary_embedding():
    from mlperf_training_b200.ops import kernels as K
    B, S, Hq, Hkv, D = 2, 10, 4, 2, 8
    mask = F.attention_mask(B, S, documents=documents(B, S, "few"))
    cos, sin = K.rope_tables(S, D, 1e4, "cpu")
    x = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1))
    do = torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(2))
    a = x.clone().requires_grad_(True)
    y = F.masked_attention_packed(a * 1.0, mask, Hq=Hq, Hkv=Hkv, D=D, cos=cos, sin=sin, softcap=5.0)
    (ga,) = torch.autograd.grad(y, a, do)
    b = x.clone().requires_grad_(True)
    r = F.rope_packed(b, cos, sin, S=S, Hq=Hq, Hkv=Hkv, D=D).view(B, S, -1)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in r.split([Hq * D, Hkv * D, Hkv * D], -1))
    z = F.masked_attention(q, k, v, mask, softcap=5.0).reshape(B * S, Hq * D)
    (gb,) = torch.autograd.grad(z, b, do)
    assert torch.allclose(y, z, rtol=1e-6, atol=1e-7) and torch.allclose(ga, gb, rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError):
        F.masked_attention_packed(x, F.attention_mask(B, 5, S), Hq=Hq, Hkv=Hkv, D=D)
    with pytest.raises(ValueError):
        F.masked_attention_packed(x[:, :-1], mask, Hq=Hq, Hkv=Hkv, D=D)


@pytest.mark.parametrize("change", [
    dict(B=0), dict(Sq=0), dict(Sq=7), dict(window=-1), dict(window=2 ** 30), dict(documents=torch.zeros(2, 5, dtype=torch.int32)),
    dict(documents=torch.zeros(2, 6)), dict(documents=torch.zeros(2, 6, dtype=torch.int32, device="meta")), dict(prefix=torch.zeros(2, 6)),
    dict(prefix=torch.zeros(2, 7, dtype=torch.bool)), dict(prefix=torch.zeros(2, 6, dtype=torch.bool), causal=False),
])
def test_mask_refusals(change):
    a = {**dict(B=2, Sq=6, Skv=6, device="cpu"), **change}
    with pytest.raises(ValueError, match="attention_mask"):
        F.attention_mask(a.pop("B"), a.pop("Sq"), a.pop("Skv"), **a)


def z(*s, **k):
    return torch.zeros(*s, **k)


@pytest.mark.parametrize("change", [
    dict(q=z(2, 6, 4)), dict(q=z(2, 6, 3, 8)), dict(q=z(2, 5, 4, 8)), dict(k=z(2, 6, 2, 4)), dict(v=z(2, 7, 2, 8)), dict(k=z(2, 7, 2, 8), v=z(2, 7, 2, 8)),
    dict(k=z(2, 6, 2, 8).half()), dict(q=z(2, 6, 4, 8, device="meta")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(scale=0.0),
    dict(scale=float("nan")), dict(slopes=z(3)), dict(slopes=z(4, dtype=torch.int32)), dict(slopes=z(4, requires_grad=True)), dict(sink=z(5)),
    dict(sink=z(4, device="meta")), dict(k=z(2, 6, 0, 8), v=z(2, 6, 0, 8)),
])
def test_refusals(change):
    a = {**dict(q=z(2, 6, 4, 8), k=z(2, 6, 2, 8), v=z(2, 6, 2, 8)), **change}
    with pytest.raises(ValueError, match="masked_attention"):
        F.masked_attention(a.pop("q"), a.pop("k"), a.pop("v"), F.attention_mask(2, 6), **a)


def test_operands_as_the_kernels_read_them():
    """Pitches of views, and copies where a view cannot be read."""
    buf = torch.zeros(2, 10, 24 * 8, dtype=torch.bfloat16)
    ok = buf[:, :, 64:128].unflatten(-1, (2, 32))
    t, row, batch = MA._bshd(ok)
    assert t is ok and (row, batch) == (192, 1920)
    for bad in (buf[:, :, 4:68].unflatten(-1, (2, 32)), ok.transpose(1, 2), ok[:, :1].expand(2, 10, 2, 32), ok[..., ::2], ok.flip(1)[:, :, :1].expand(2, 10, 2, 32)):
        t, row, batch = MA._bshd(bad)
        assert t.is_contiguous() and row == bad.shape[2] * bad.shape[3] and batch == row * bad.shape[1] and torch.equal(t, bad)
    one = buf[:1, :1, :64].unflatten(-1, (2, 32))
    assert MA._bshd(one)[1:] == (64, 64)
