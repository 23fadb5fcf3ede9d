"""Masked attention kernels against the definition in 64 bits: masks as the kernels have them, output and gradients over mask kinds, score
forms, head layouts, lengths from one token on, strides; rows that see nothing; padding; streams, graphs."""
import pytest
import torch

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F
from mlperf_training_b200.ops import masked_attention as MA
from tests import masked_oracle as O
from tests.test_masked_attention import KINDS, MASKS, SCORES, documents, flags, make, tensors

pytestmark = pytest.mark.gpu


def to(kw, dev="cuda"):
    return {n: v.to(dev) if torch.is_tensor(v) else v for n, v in kw.items()}


@pytest.mark.parametrize("m", MASKS + [dict(window=200), dict(prefix=True, window=700)], ids=str)
@pytest.mark.parametrize("kind", KINDS + ["absent"])
@pytest.mark.parametrize("B,Sq,Skv", [(1, 1, 1), (2, 40, 40), (3, 129, 129), (1, 1, 300), (2, 300, 1111), (1, 9001, 9001), (2, 130, 4097), (1, 20000, 20000),
                                        (2, 300, 49153)])
def test_masks(B, Sq, Skv, kind, m):
    """The kernels' intervals against the CPU's, and the tables of tiles against the intervals."""
    kw = make(B, Sq, Skv, kind, m)
    ref = F.attention_mask(B, Sq, Skv, **kw)
    mask = F.attention_mask(B, Sq, Skv, **to(kw), device="cuda")
    Sp, Kp = -(-Sq // 256) * 256, -(-Skv // 128) * 128
    nq, nk = Sp // 128, Kp // 128
    buf = mask.buf.cpu()
    cut = [0]

    def take(n, *shape):
        cut[0] += n
        return buf[cut[0] - n:cut[0]].view(*shape)

    qt, kt = take(B * nq * 4, B, nq, 4), take(B * nk * 4, B, nk, 4)
    q_iv, k_iv = take(B * Sp * 2, B, Sp, 2), take(B * Kp * 2, B, Kp, 2)
    oq, ok = take(B * nq // 2, -1), take(B * nk, -1)
    # (a bit of each query tile says whether some key of its sequence is seen by no query)
    unseen = (k_iv[:, :Skv, 0] >= k_iv[:, :Skv, 1]).any(1)
    assert torch.equal((qt[..., 1] >> 30) != 0, unseen[:, None].expand(B, nq))
    qt = torch.stack([qt[..., 0], qt[..., 1] & ~(1 << 30), qt[..., 2], qt[..., 3]], -1)
    lo, hi = q_iv[:, :Sq, 0], q_iv[:, :Sq, 1]
    assert torch.equal(lo, ref.lo.int()) and torch.equal(hi, ref.hi.int())
    assert (lo[:, 1:] >= lo[:, :-1]).all() and (hi[:, 1:] >= hi[:, :-1]).all()       # what the tile ranges rest on
    if Sq * Skv <= 1 << 21:
        see = ref.visible()
        qs = torch.arange(Sq)
        assert torch.equal((qs[None, :, None] >= k_iv[:, None, :Skv, 0]) & (qs[None, :, None] < k_iv[:, None, :Skv, 1]), see)
    for iv, tiles, rows in ((q_iv, qt, Sq), (k_iv, kt, Skv)):
        for b in range(B):
            for t in range(tiles.shape[1]):
                v = iv[b, t * 128:min((t + 1) * 128, rows)]
                live = v[v[:, 0] < v[:, 1]]
                want = (int(live[:, 0].min()) // 128, -(-int(live[:, 1].max()) // 128)) if len(live) else (0, 0)
                assert tuple(tiles[b, t, :2].tolist()) == want
                a, c = tiles[b, t, 2:].tolist()
                if len(v) and a < c:                                # [a, c) is visible to every row of the tile
                    assert (v[:, 0] <= a).all() and (v[:, 1] >= c).all()
    pair = qt.view(B, nq // 2, 2, 4)
    n = (pair[..., 1] - pair[..., 0]).sum(-1)
    shared = (pair[..., 1].amin(-1) - pair[..., 0].amax(-1)).clamp(min=0)
    cost = (4 * (n - shared) + shared).flatten()
    assert torch.equal(oq.sort()[0], torch.arange(B * nq // 2).int()) and (cost[oq.long()].diff() <= 0).all()
    cost = (kt[..., 1] - kt[..., 0]).flatten()
    assert torch.equal(ok.sort()[0], torch.arange(B * nk).int()) and (cost[ok.long()].diff() <= 0).all()
    assert torch.equal(mask.visible().cpu(), ref.visible())


def oracle(q, k, v, do, ok, kw):
    """On the GPU in 64 bits, all heads at once."""
    ins = [t.detach().cuda().double().requires_grad_(True) for t in (q, k, v)]
    sink = kw["sink"].cuda().double().requires_grad_(True) if kw.get("sink") is not None else None
    ok, (B, Sq, Hq, D), Skv = ok.cuda(), q.shape, k.shape[1]
    qd, kd, vd = ins[0].transpose(1, 2), *(t.transpose(1, 2).repeat_interleave(Hq // k.shape[2], 1) for t in ins[1:])
    s = qd @ kd.mT * (kw.get("scale") or D ** -0.5)
    if kw.get("softcap"):
        s = kw["softcap"] * torch.tanh(s / kw["softcap"])
    if kw.get("slopes") is not None:
        at = torch.arange(Skv, device="cuda").double()
        s = s - kw["slopes"].cuda().double()[:, None, None] * (at[Skv - Sq:, None] - at).abs()
    s = s.masked_fill(~ok[:, None], -torch.inf)
    if sink is not None:
        s = torch.cat([s, sink.view(1, -1, 1, 1).expand(B, -1, Sq, 1)], -1)
    live = (s > -torch.inf).any(-1, keepdim=True)
    p = torch.where(live, torch.softmax(torch.where(live, s, 0.0), -1), 0.0)[..., :Skv]
    y = (p @ vd).transpose(1, 2)
    return [y.detach()] + list(torch.autograd.grad(y, ins + ([sink] if sink is not None else []), do.cuda().double()))


def close(got, want, rel, what):
    """Relative to the whole tensor's size, and element by element to 30 times that of its rms."""
    d, n = (got.double() - want).norm(), want.norm()
    assert torch.isfinite(got.double()).all(), what
    assert d <= rel * n + 1e-30, f"{what}: {float(d / n):.2e} of {rel:.1e}"
    assert (got.double() - want).abs().max() <= 30 * rel * torch.maximum(want.abs().max(), n / want.numel() ** 0.5) + 1e-30, what


# Output: P rounded to bf16 (2^-9 rms at most a key, averaged over keys), O rounded once (2^-9 / sqrt 3 rms): below 2^-8 together.  dV: P and
# dO as P's rounding, then dV's: the same.  dQ, dK: P's exponent (lse 2^-9 / sqrt 3), dS rounded (the same) and the result's rounding, where
# dS is a difference whose terms are kept to 2^-17: below 2^-7 even for rows of few keys.  The cap's polynomial (7e-6 of a score) is inside.
OUT, GRAD = 2 ** -8, 2 ** -7


def run(q, k, v, do, mask, s, dev="cuda"):
    ins = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    s = to(s)
    if "sink" in s:
        ins.append(s["sink"].requires_grad_(True))
    y = F.masked_attention(*ins[:3], mask, **s)
    return [y.detach()] + list(torch.autograd.grad(y, ins, do.to(dev)))


def check(B, Sq, Skv, Hq, Hkv, D, kind, m, score):
    kw = make(B, Sq, Skv, kind, m)
    mask = F.attention_mask(B, Sq, Skv, **to(kw), device="cuda")
    q, k, v, do, s = tensors(B, Sq, Skv, Hq, Hkv, D, score, torch.bfloat16)
    ok = F.attention_mask(B, Sq, Skv, **kw).visible()
    want = oracle(q, k, v, do, ok, s)
    got = run(q, k, v, do, mask, s)
    _lib.check_status("masked attention")
    # sums whose terms cancel to nothing (rows of one key have no gradient of q and k): compared to the size of the terms
    for name, a, b, r in zip(("out", "dq", "dk", "dv", "dsink"), got, want, (OUT, GRAD, GRAD, OUT, GRAD)):
        if name in ("dq", "dk") and (ok.sum(-1) <= 1).all() and "sink" not in s:
            assert a.abs().max() <= 2 ** -7 * float(do.norm(dim=-1).max() * v.norm(dim=-1).max() * max(k.norm(dim=-1).max(), q.norm(dim=-1).max())) / D ** 0.5
            continue
        close(a, b, r, name)
    empty = ~ok.any(-1)
    assert (got[0].cpu()[empty] == 0).all() and (got[1].cpu()[empty] == 0).all()
    unseen = ~ok.any(1)
    assert (got[2].cpu()[unseen] == 0).all() and (got[3].cpu()[unseen] == 0).all()
    # without a gradient: few rows a key head take a kernel of their own, others sum their rows before the probabilities are rounded
    with torch.no_grad():
        y = F.masked_attention(*(t.cuda() for t in (q, k, v)), mask, **to(s))
    close(y, want[0], OUT, "out without a gradient")
    assert (y.cpu()[empty] == 0).all()
    _lib.check_status("masked attention")
    return got


@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind,m", [("left", MASKS[0]), ("holes", MASKS[4]), ("few", MASKS[1]), ("few", dict(window=100))], ids=str)
def test_few_rows_over_many_keys(D, kind, m, score):
    """Keys split over several blocks (joined by a second launch), rows of several documents."""
    for B, Sq, Skv, Hq, Hkv in ((2, 1, 5000, 8, 2), (1, 7, 2311, 9, 1), (3, 3, 777, 4, 4), (1, 16, 4097, 4, 1)):
        kw = make(B, Sq, Skv, kind, m)
        mask = F.attention_mask(B, Sq, Skv, **to(kw), device="cuda")
        q, k, v, do, s = tensors(B, Sq, Skv, Hq, Hkv, D, score, torch.bfloat16)
        ok = F.attention_mask(B, Sq, Skv, **kw).visible()
        want = oracle(q, k, v, do, ok, s)[0]
        pad = ~ok.any(1)                                       # keys that nothing sees may hold anything
        k[pad], v[pad] = float("nan"), float("inf")
        with torch.no_grad():
            out, lse, _ = MA.masked_attention_fwd(*(t.cuda() for t in (q, k, v)), mask, **to(s))
        close(out, want, OUT, "out")
        assert (out.cpu()[~ok.any(-1)] == 0).all()
        _lib.check_status("few rows")


@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind,m", [("few", MASKS[0]), ("holes", MASKS[4])], ids=str)
def test_scores(D, kind, m, score):
    check(2, 333, 333, 4, 2, D, kind, m, score)


@pytest.mark.parametrize("m", MASKS + [dict(window=150), dict(causal=False, window=150)], ids=str)
@pytest.mark.parametrize("kind", KINDS + ["absent"])
def test_mask_kinds(kind, m):
    check(3, 517, 517, 2, 1, 64, kind, m, SCORES[0])


@pytest.mark.parametrize("S", [1, 2, 7, 31, 64, 127, 128, 129, 255, 256, 257, 384, 640])
@pytest.mark.parametrize("kind", ["one", "few", "padded"])
def test_lengths(S, kind):
    check(2, S, S, 4, 4, 128, kind, MASKS[0], SCORES[0])


@pytest.mark.parametrize("Sq,Skv", [(1, 2), (1, 1000), (3, 129), (60, 700), (130, 4097), (200, 201)])
@pytest.mark.parametrize("kind", ["one", "left", "few"])
@pytest.mark.parametrize("score", [SCORES[0], SCORES[3]], ids=str)
def test_last_positions(Sq, Skv, kind, score):
    check(2, Sq, Skv, 8, 2, 128, kind, MASKS[0], score)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (5, 1), (12, 4), (16, 1)])
def test_head_layouts(Hq, Hkv):
    check(2, 200, 200, Hq, Hkv, 64, "few", MASKS[0], SCORES[2])


@pytest.mark.parametrize("score", SCORES[:4], ids=str)
def test_long_rows(score):
    check(1, 3001, 3001, 4, 2, 128, "few", MASKS[0], score)


@pytest.mark.parametrize("score", SCORES, ids=str)
@pytest.mark.parametrize("kind,m", [("one", MASKS[0]), ("few", MASKS[1]), ("holes", MASKS[4]), ("left", dict(window=700)), ("few", dict(causal=False))], ids=str)
@pytest.mark.parametrize("Sq,Skv,Hq,Hkv,D", [(2311, 2311, 2, 1, 64), (300, 5003, 4, 2, 128)])
def test_few_tiles_over_many_keys(Sq, Skv, Hq, Hkv, D, kind, m, score):
    """Key tiles of a pair of query tiles in parts (forward) and steps of a key tile shared (backward), beside pairs and tiles that stay whole."""
    assert _lib.load().b200_attn_masked_fwd_workspace(1, Sq, Skv, Hq, D) > 0
    check(1, Sq, Skv, Hq, Hkv, D, kind, m, score)


def test_padding_may_hold_anything_beside_parts():
    B, S = 1, 3000
    ids = documents(B, S, "padded")
    q, k, v, do, s = tensors(B, S, S, 2, 2, 64, {}, torch.bfloat16)
    ok = F.attention_mask(B, S, documents=ids).visible()
    want = oracle(q, k, v, do, ok, s)[0]
    pad = ~ok.any(1)
    assert pad.any()
    q[pad], k[pad], v[pad] = float("inf"), float("nan"), float("nan")
    with torch.no_grad():
        y = F.masked_attention(q.cuda(), k.cuda(), v.cuda(), F.attention_mask(B, S, documents=ids.cuda()))
    close(y, want, OUT, "out")
    assert (y.cpu()[~ok.any(-1)] == 0).all()
    _lib.check_status("parts")


@pytest.mark.parametrize("cap", [0.25, 1.0, 30.0])
def test_scores_far_beyond_the_cap(cap):
    """Scores of standard deviation 12 and more: both forms of the tangent."""
    mask = F.attention_mask(2, 300, documents=documents(2, 300, "few").cuda())
    q, k, v, do, _ = tensors(2, 300, 300, 4, 2, 64, {}, torch.bfloat16)
    q = (q * 12).bfloat16()
    want = oracle(q, k, v, do, mask.visible().cpu(), {"softcap": cap})
    for name, a, b, r in zip(("out", "dq", "dk", "dv"), run(q, k, v, do, mask, {"softcap": cap}), want, (OUT, GRAD, GRAD, OUT)):
        close(a, b, r, name)


def test_one_dominant_key():
    """Near-one-hot rows, whose dS is a small difference: scores of standard deviation 8."""
    mask = F.attention_mask(1, 400, device="cuda")
    q, k, v, do, _ = tensors(1, 400, 400, 4, 2, 64, {}, torch.bfloat16)
    q = (q * 8).bfloat16()
    for name, a, b, r in zip(("out", "dq", "dk", "dv"), run(q, k, v, do, mask, {}), oracle(q, k, v, do, mask.visible().cpu(), {}), (OUT, GRAD, GRAD, OUT)):
        close(a, b, r, name)


def test_padding_may_hold_anything_in_the_forward_pass():
    S = 700
    ids = documents(2, S, "holes")
    ids[0, 128:256] = -1
    ids[1, 600:] = -1
    mask = F.attention_mask(2, S, documents=ids.cuda())
    q, k, v, _, _ = (t.cuda() if torch.is_tensor(t) else t for t in tensors(2, S, S, 4, 2, 128, {}, torch.bfloat16))
    ref = F.masked_attention(q, k, v, mask)
    pad = (ids < 0).cuda()
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[pad] = bad
    assert torch.equal(F.masked_attention(q, k, v, mask), ref)
    v[pad] = float("-inf")
    assert torch.equal(F.masked_attention(q, k, v, mask, softcap=5.0), F.masked_attention(q, k, torch.where(pad[..., None, None], 0, v), mask, softcap=5.0))
    _lib.check_status("padding")


@pytest.mark.parametrize("off", [0, 8, 3])
def test_views_of_a_packed_buffer(off):
    B, S, Hq, Hkv, D = 2, 150, 4, 2, 64
    mask = F.attention_mask(B, S, documents=documents(B, S, "few").cuda())
    q, k, v, do, _ = (t.cuda() if torch.is_tensor(t) else t for t in tensors(B, S, S, Hq, Hkv, D, {}, torch.bfloat16))
    ref = run(q, k, v, do, mask, {})
    buf = torch.zeros(B, S, (Hq + 2 * Hkv) * D + 40, device="cuda", dtype=torch.bfloat16)
    buf[..., off:off + (Hq + 2 * Hkv) * D] = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    buf.requires_grad_(True)
    qkv = buf[..., off:off + (Hq + 2 * Hkv) * D]
    a, b, c = (t.unflatten(-1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    y = F.masked_attention(a, b, c, mask)
    (g,) = torch.autograd.grad(y, buf, do.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(y.detach(), ref[0])
    g = g[..., off:off + (Hq + 2 * Hkv) * D].split([Hq * D, Hkv * D, Hkv * D], -1)
    # (dQ is added up in another order each time; dK and dV are not)
    assert torch.equal(g[1].reshape(ref[2].shape), ref[2]) and torch.equal(g[2].reshape(ref[3].shape), ref[3])
    close(g[0].reshape(ref[1].shape), ref[1].double(), 2 ** -8, "dq")
    with torch.no_grad():
        plain = F.masked_attention(q, k, v, mask)
        assert torch.equal(F.masked_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k.expand(B, S, Hkv, D), v, mask), plain)
        assert torch.equal(F.masked_attention(a, b, c, mask), plain)
    _lib.check_status("views")


def test_shared_keys_of_a_batch():
    """Keys broadcast over the batch get the sum of its gradients."""
    B, S = 3, 130
    mask = F.attention_mask(B, S, device="cuda")
    q, k, v, do, _ = tensors(B, S, S, 4, 2, 64, {}, torch.bfloat16)
    k1, v1 = k[:1].cuda().requires_grad_(True), v[:1].cuda().requires_grad_(True)
    y = F.masked_attention(q.cuda(), k1.expand(B, -1, -1, -1), v1.expand(B, -1, -1, -1), mask)
    got = torch.autograd.grad(y, [k1, v1], do.cuda())
    want = oracle(q, k[:1].expand_as(k), v[:1].expand_as(v), do, mask.visible().cpu(), {})
    close(got[0], want[2].sum(0, keepdim=True), GRAD, "dk")
    close(got[1], want[3].sum(0, keepdim=True), GRAD, "dv")


def test_packed_form():
    B, S, Hq, Hkv, D = 2, 200, 4, 2, 64
    from mlperf_training_b200.ops import kernels as K
    ids = documents(B, S, "few")
    out = []
    x = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).bfloat16()
    do = torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(2)).bfloat16()
    for dev in ("cpu", "cuda"):
        cos, sin = K.rope_tables(S, D, 1e4, dev)
        a = x.to(dev).requires_grad_(True)
        y = F.masked_attention_packed(a * 1.0, F.attention_mask(B, S, documents=ids.to(dev)), Hq=Hq, Hkv=Hkv, D=D, cos=cos, sin=sin, softcap=5.0)
        out.append([y.detach().cpu().double(), torch.autograd.grad(y, a, do.to(dev))[0].cpu().double()])
    # both round q and k after the rotation to bf16, the CPU in other places
    close(out[1][0], out[0][0], 2 * OUT, "out")
    close(out[1][1], out[0][1], 2 * GRAD, "dqkv")
    _lib.check_status("packed")


def test_captured_and_replayed_beside_an_eager_call():
    B, S = 2, 300
    ids = documents(B, S, "few").cuda()
    q, k, v, do, _ = (t.cuda() if torch.is_tensor(t) else t for t in tensors(B, S, S, 4, 2, 64, {}, torch.bfloat16))
    F.masked_attention(q, k, v, F.attention_mask(B, S, documents=ids))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.masked_attention(q, k, v, F.attention_mask(B, S, documents=ids), softcap=10.0)
    for seed in (1, 2):
        ids.copy_(documents(B, S, "holes", seed))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            want = F.masked_attention(q, k, v, F.attention_mask(B, S, documents=ids), softcap=10.0)
            torch.cuda.current_stream().synchronize()
        assert torch.equal(y, want)
    _lib.check_status("graph")


def test_mask_of_very_many_positions():
    Skv = 2 ** 28 + 5
    m = F.attention_mask(1, 1, Skv, window=700, device="cuda")
    nk, Kp = -(-Skv // 128), -(-Skv // 128) * 128
    at = 2 * 4 + nk * 4                                        # query tiles, key tiles; then keys of the queries, queries of the keys, the orders
    assert m.buf[at:at + 2].tolist() == [Skv - 700, Skv]
    order = m.buf[at + 2 * 256 + 2 * Kp + 1:][:nk].long()
    assert torch.equal(order.sort()[0], torch.arange(nk, device="cuda"))
    seen = range((Skv - 700) // 128, nk)                       # come first
    assert set(order[:len(seen)].tolist()) == set(seen)
    _lib.check_status("mask")


def test_refuses_what_the_kernels_do_not_read():
    mask = F.attention_mask(1, 4, device="cuda")
    x = torch.zeros(1, 4, 2, 64, device="cuda")
    for bad in (x, x.half(), torch.zeros(1, 4, 2, 32, device="cuda", dtype=torch.bfloat16), torch.zeros(1, 4, 2, 256, device="cuda", dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            F.masked_attention(bad, bad, bad, mask)
    b = x.bfloat16()
    with pytest.raises(ValueError):
        F.masked_attention(b, b, b, F.attention_mask(1, 4))              # a mask of the CPU
    with pytest.raises(ValueError):
        F.attention_mask(1, 4, documents=torch.zeros(1, 4, dtype=torch.int32), device="cuda")
