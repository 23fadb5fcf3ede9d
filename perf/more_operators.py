"""Operators of post-training on packed documents, one pass each, on one GPU: attention with document, prefix and window
masks, capped scores and a distance bias; routing to experts; distillation from a teacher's top logits.

A case is a dict of plain values; ``kind`` says which operator it takes:

    attn     attention of the last Sq of Skv positions (mask made from document ids and prefix flags, then the attention),
             optionally with its backward pass
    route    routing of T tokens to k of E experts (softmax or sigmoid scores, a bias that only selects, groups of experts),
             optionally with the gradient of the logits and the step of the bias
    distill  loss against a teacher's K largest logits mixed with cross-entropy, optionally with the gradient of the logits

``listed()`` are fixed sizes, ``draw(rng)`` gives others of the same ranges.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
RATE = 1e-3            # step of a router's balance bias
SCALE = 2.5            # factor of its weights


# --------------------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------------------
def _attn(B, Sq, Skv, Hq, Hkv, D, docs=0, pad=0, prefix=False, causal=True, window=0, softcap=0.0, alibi=False, train=False, **more):
    return dict(kind="attn", B=B, Sq=Sq, Skv=Skv, Hq=Hq, Hkv=Hkv, D=D, docs=docs, pad=pad, prefix=prefix, causal=causal, window=window,
                softcap=softcap, alibi=alibi, train=train, **more)


def _route(T, E, k, score, bias=False, groups=1, top_groups=1, renormalize=True, dtype="f32", train=False, **more):
    return dict(kind="route", T=T, E=E, k=k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalize=renormalize,
                dtype=dtype, train=train, **more)


def _distill(T, V, K, alpha, temperature, rest=False, dtype="bf16", train=False, **more):
    return dict(kind="distill", T=T, V=V, K=K, alpha=alpha, temperature=temperature, rest=rest, dtype=dtype, train=train, **more)


def listed():
    return [
        # a short prompt through a small decoder's layer: launches are most of the time
        _attn(1, 61, 61, 8, 2, 64, docs=2, name="attn_short"),
        # generation: the next token of eight sequences of unlike lengths, padded on the left
        _attn(8, 1, 16384, 32, 8, 128, pad=9000, softcap=30.0, name="attn_token"),
        # evaluation of packed documents with a window and a distance bias, an odd length, heads of 64
        _attn(2, 4001, 4001, 64, 8, 64, docs=9, pad=70, window=1024, alibi=True, name="attn_window"),
        # fine-tuning on packed prompts and answers: prompts see themselves both ways, scores are capped
        _attn(4, 2048, 2048, 32, 8, 128, docs=6, pad=200, prefix=True, softcap=50.0, train=True, name="attn_prefix_train"),
        # an 8B decoder's layer in training: a sequence of 8192 packed from five documents
        _attn(1, 8192, 8192, 32, 8, 128, docs=5, train=True, name="attn_docs_train"),
        # a handful of tokens through a router of 32 experts
        _route(7, 32, 4, "softmax", name="route_token"),
        # training of 8192 tokens, experts in groups, sigmoid scores and a balance bias
        _route(8192, 64, 6, "sigmoid", bias=True, groups=8, top_groups=4, train=True, name="route_groups_train"),
        # eight sequences of 8192 through a router of 256 experts, bf16 logits
        _route(65536, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, dtype="bf16", train=True, name="route_large_train"),
        # a few tokens against a small vocabulary
        _distill(5, 2048, 16, 0.5, 2.0, train=True, name="distill_rows"),
        # evaluation against the teacher on an odd number of tokens, logits in 32 bits
        _distill(1027, 32000, 64, 0.9, 1.0, dtype="f32", name="distill_eval"),
        # training against the teacher's 64 largest logits and the labels, a vocabulary of 128256
        _distill(8192, 128256, 64, 0.7, 2.0, train=True, name="distill_train"),
        # training with the rest of the vocabulary as one more event, a vocabulary of 201088
        _distill(2048, 201088, 32, 1.0, 1.0, rest=True, train=True, name="distill_rest_train"),
    ]


def _log(rng, lo, hi, step=1):
    """An integer between lo and hi, spread over its logarithm, rounded to a multiple of ``step``."""
    v = int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    return max(step, min(hi, max(lo, v)) // step * step)


def draw(rng):
    kind = rng.choice(["attn", "attn", "route", "distill"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if kind == "attn":
        D, Hkv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        extra = dict(softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=flag())
        if rng.random() < 0.3:       # a few new positions behind a long past
            Skv, B = _log(rng, 1, 32768), _log(rng, 1, 16)
            return _attn(B, min(Skv, rng.choice([1, 1, 1, 2, 5])), Skv, Hq, Hkv, D, pad=rng.randrange(Skv), window=rng.choice([0, 0, _log(rng, 1, 4096)]),
                         **extra)
        most = max(work(c)["flops"] for c in listed())
        train = flag()           # trained sequences have some tokens: a row that sees one key alone has no gradient to compare
        S = _log(rng, 24 if train else 1, math.isqrt(32 * 8192 * 8192 // max(32, Hq)))
        B = _log(rng, 1, max(1, min(16, 32 * 8192 * 8192 // (Hq * S * S))))
        causal = rng.random() < 0.8
        c = _attn(B, S, S, Hq, Hkv, D, docs=rng.choice([0, _log(rng, 1, 24 if S > 400 else 1 + S // 8)]),
                  pad=rng.choice([0, rng.randrange(S // 2 + 1)]), causal=causal, prefix=causal and flag(),
                  window=rng.choice([0, 0, _log(rng, 16 if train else 1, 2048)]), train=train, **extra)
        while work(c)["flops"] > most:
            S = S * 7 // 8
            c.update(Sq=S, Skv=S, pad=min(c["pad"], S // 2))
        return c
    if kind == "route":
        G = rng.choice([1, 1, 4, 8])
        E = G * _log(rng, 2, 256 // G)
        top = rng.randint(max(1, G // 2), G)
        k = rng.randint(1, min(16, top * (E // G)))
        return _route(_log(rng, 1, 65536), E, k, rng.choice(["softmax", "sigmoid"]), bias=flag(), groups=G, top_groups=top,
                      renormalize=k > 1 and flag(), dtype=rng.choice(["f32", "bf16"]), train=flag())
    V = _log(rng, 64, 201088)
    rest = rng.random() < 0.3
    return _distill(_log(rng, 1, max(1, min(16384, 8192 * 128256 // V))), V, _log(rng, 1, min(128, V // 2)), rng.choice([1.0, 0.9, 0.5]),
                    1.0 if rest else rng.choice([1.0, 2.0, 4.0]), rest=rest, dtype=rng.choice(["bf16", "bf16", "f32"]), train=flag())


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _layout(case):
    """For each sequence its documents as (start, end, end of the prefix); other positions are padding.  Sequences of several
    positions at a time are padded at their end, those whose last positions alone are asked at their start."""
    B, S, n, rows = case["B"], case["Skv"], case["docs"], []
    r = random.Random(B * 1000003 + S * 101 + n)
    for b in range(B):
        pad = min(case["pad"] * (b + 1) // B, S - 1) if case["pad"] else 0
        lo, hi = (pad, S) if case["Sq"] < S else (0, S - pad)
        cuts = sorted(r.sample(range(lo + 1, hi), min(max(n, 1), hi - lo) - 1))
        ends = cuts + [hi]
        rows.append([(s, e, s + (r.randint(0, e - s) if case["prefix"] else 0)) for s, e in zip([lo] + cuts, ends)])
    return rows


def _ids_and_flags(case):
    ids = torch.full((case["B"], case["Skv"]), -1, dtype=torch.int32)
    flags = torch.zeros(case["B"], case["Skv"], dtype=torch.bool)
    for b, row in enumerate(_layout(case)):
        for n, (s, e, p) in enumerate(row):
            ids[b, s:e] = n
            flags[b, s:p] = True
    return ids.to(DEV), flags.to(DEV)


def _teacher(g, T, V, K, rest):
    """Each token's K likeliest of V for a teacher, distinct, and their logits (``rest``: log-probabilities, some left over)."""
    at = torch.randint(0, V, (T, 1), generator=g, device=DEV)
    ids = (at + torch.arange(K, device=DEV) * (V // K)) % V
    val = torch.sort(4 * torch.randn(T, K, generator=g, device=DEV), -1, descending=True)[0]
    if rest:
        left = val.amax(-1, keepdim=True) + 3 * torch.randn(T, 1, generator=g, device=DEV) - 3
        val = torch.log_softmax(torch.cat([val, left], -1).double(), -1)[:, :K].float()
    return ids, val


def prepare(case, seed):
    g, s = _gen(seed), dict(case)
    if case["kind"] == "attn":
        B, Sq, Skv, Hq, Hkv, D, t = (case[n] for n in ("B", "Sq", "Skv", "Hq", "Hkv", "D", "train"))
        s["q"] = torch.randn(B, Sq, Hq, D, generator=g, device=DEV).mul_(1.5).to(BF16).requires_grad_(t)
        s["k"] = torch.randn(B, Skv, Hkv, D, generator=g, device=DEV).mul_(1.5).to(BF16).requires_grad_(t)
        s["v"] = torch.randn(B, Skv, Hkv, D, generator=g, device=DEV).to(BF16).requires_grad_(t)
        s["dout"] = torch.randn(B, Sq, Hq, D, generator=g, device=DEV).mul_(1e-2).to(BF16) if t else None
        s["documents"] = s["flags"] = s["slopes"] = None
        if case["docs"] or case["pad"]:
            s["documents"], s["flags"] = _ids_and_flags(case)
        elif case["prefix"]:
            s["flags"] = _ids_and_flags(case)[1]
        if case["alibi"]:
            s["slopes"] = torch.exp2(-8 * torch.arange(1, Hq + 1, device=DEV).float() / Hq)
    elif case["kind"] == "route":
        T, E = case["T"], case["E"]
        s["logits"] = (torch.randn(T, E, generator=g, device=DEV) + 0.5 * torch.randn(E, generator=g, device=DEV))
        s["logits"] = s["logits"].to(BF16 if case["dtype"] == "bf16" else torch.float32).requires_grad_(case["train"])
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
        s["gw"] = torch.randn(T, case["k"], generator=g, device=DEV) * 1e-2 if case["train"] else None
    else:
        T, V, K = case["T"], case["V"], case["K"]
        s["ids"], s["values"] = _teacher(g, T, V, K, case["rest"])
        z = torch.randn(T, V, generator=g, device=DEV).mul_(2)
        # a student that has learned some of it
        z.scatter_add_(1, s["ids"], 6 + 0.5 * (s["values"] - s["values"].amax(-1, keepdim=True)))
        s["logits"] = z.to(BF16 if case["dtype"] == "bf16" else torch.float32).requires_grad_(case["train"])
        labels = torch.where(torch.rand(T, generator=g, device=DEV) < 0.8, s["ids"][:, 0], torch.randint(0, V, (T,), generator=g, device=DEV))
        s["labels"] = torch.where(torch.rand(T, generator=g, device=DEV) < 0.1, -100, labels)
        s["gy"] = (0.5 + torch.rand(T, generator=g, device=DEV)) / T if case["train"] else None
    return s


# --------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# --------------------------------------------------------------------------------------
def _visible(s):
    """[B, Sq, Skv]: which keys a query sees."""
    B, Sq, Skv = s["B"], s["Sq"], s["Skv"]
    at = torch.arange(Skv, device=DEV)
    p, k = at[Skv - Sq:, None], at[None, :]
    past = (k <= p).expand(B, Sq, Skv) if s["causal"] else torch.ones(B, Sq, Skv, dtype=torch.bool, device=DEV)
    ids = s["documents"] if s["documents"] is not None else torch.zeros(B, Skv, dtype=torch.int32, device=DEV)
    if s["prefix"]:
        # a key belongs to the prefix if it and all before it in its document are flagged
        new = torch.ones_like(ids, dtype=torch.bool)
        new[:, 1:] = ids[:, 1:] != ids[:, :-1]
        start = torch.cummax(torch.where(new, at, 0), -1)[0]
        bare = torch.cumsum((~s["flags"]).int(), -1)
        before = bare.gather(1, start) - (~s["flags"]).int().gather(1, start)
        past = past | (bare == before)[:, None, :]
    ok = past & (ids[:, Skv - Sq:, None] == ids[:, None, :]) & (ids >= 0)[:, None, :]
    return ok & (p - k < s["window"]) if s["window"] else ok


def _plain_attn(s):
    group, D = s["Hq"] // s["Hkv"], s["D"]
    q = s["q"].float().transpose(1, 2)
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(group, 1) for n in ("k", "v"))
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(D))
    if s["softcap"]:
        x = x.div_(s["softcap"]).tanh_()
        slope_of_cap = x
        x = x * s["softcap"]
    if s["slopes"] is not None:
        at = torch.arange(s["Skv"], device=DEV, dtype=torch.float32)
        x = x - s["slopes"][:, None, None] * (at[s["Skv"] - s["Sq"]:, None] - at).abs()
    x = x.masked_fill_(~_visible(s)[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    out = {"out": torch.matmul(p, v).transpose(1, 2).to(BF16)}
    if s["train"]:
        do = s["dout"].float().transpose(1, 2)
        shared = lambda t: t.unflatten(1, (s["Hkv"], group)).sum(2).transpose(1, 2).to(BF16)  # noqa: E731
        out["dv"] = shared(torch.matmul(p.transpose(-1, -2), do))
        dp = torch.matmul(do, v.transpose(-1, -2))
        dx = p * dp.sub_((p * dp).sum(-1, keepdim=True))
        if s["softcap"]:
            dx = dx.mul_(1 - slope_of_cap * slope_of_cap)
        dx = dx.mul_(1 / math.sqrt(D))
        out["dq"] = torch.matmul(dx, k).transpose(1, 2).to(BF16)
        out["dk"] = shared(torch.matmul(dx.transpose(-1, -2), q))
    return out


def _plain_route(s):
    T, E, k, G = s["T"], s["E"], s["k"], s["groups"]
    # in 64 bits: experts are compared by values that may lie next to each other
    x = s["logits"].double()
    score = torch.sigmoid(x) if s["score"] == "sigmoid" else torch.softmax(x, -1)
    by = score if s["bias"] is None else score + s["bias"].double()
    if s["top_groups"] < G:
        groups = by.unflatten(1, (G, E // G)).sort(-1, descending=True)[0][..., :2].sum(-1)
        kept = torch.zeros(T, G, dtype=torch.bool, device=DEV)
        kept.scatter_(1, groups.sort(dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]], True)
        by = by.masked_fill(~kept.repeat_interleave(E // G, 1), -math.inf)
    idx = by.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    picked = score.gather(1, idx)
    total = picked.sum(-1, keepdim=True) + 1e-20 if s["renormalize"] else torch.ones(T, 1, dtype=torch.float64, device=DEV)
    w = SCALE * picked / total
    counts = torch.bincount(idx.flatten(), minlength=E)
    out = {"idx": idx.int(), "w": w.float(), "counts": counts.int()}
    if s["train"]:
        dw = SCALE * s["gw"].double()
        dp = (dw - (dw * picked).sum(-1, keepdim=True) / total) / total if s["renormalize"] else dw
        if s["score"] == "sigmoid":
            dx = torch.zeros_like(score).scatter_(1, idx, dp * picked * (1 - picked))
        else:
            dx = torch.zeros_like(score).scatter_(1, idx, dp)
            dx = score * (dx - (dx * score).sum(-1, keepdim=True))
        out["dlogits"] = dx.to(s["logits"].dtype)
        if s["bias"] is not None:
            out["bias"] = (s["bias"].double() + RATE * torch.sign(counts.sum() - E * counts)).float()
    return out


def _log_sum(x):
    m = x.amax(-1, keepdim=True)
    return (x - m).exp_().sum(-1, keepdim=True).log() + m


def _plain_distill(s):
    z, ids, a, tau = s["logits"].float(), s["ids"], s["alpha"], s["temperature"]
    live = (s["labels"] != -100)[:, None]
    label = s["labels"].clamp(min=0)[:, None]
    u = z if tau == 1 else z / tau
    norm_u = _log_sum(u)
    norm_z = norm_u if tau == 1 else _log_sum(z)
    t = s["values"].double()
    logp = t if s["rest"] else t / tau - torch.logsumexp(t / tau, -1, keepdim=True)
    p = logp.exp()
    kl = (p * (logp - u.gather(1, ids) + norm_u)).sum(-1, keepdim=True)
    if s["rest"]:
        r = (1 - p.sum(-1, keepdim=True)).clamp(min=0)
        others = _log_sum(u.scatter(1, ids, -math.inf)) - norm_u
        kl = kl + torch.where(r > 0, r * (r.log() - others), 0.0)
    loss = a * tau * tau * kl + (1 - a) * (norm_z - z.gather(1, label))
    out = {"loss": torch.where(live, loss, 0.0)[:, 0].float()}
    if s["train"]:
        gy = torch.where(live, s["gy"][:, None], 0.0)
        q = (u - norm_u).exp_()
        if s["rest"]:
            g = q * ((1 - r / others.double().exp()).float())
            g.scatter_(1, ids, q.gather(1, ids))
        else:
            g = q
        g = g.scatter_add_(1, ids, -p.float()).mul_(a * tau * gy)
        if a < 1:
            g = g.add_((z - norm_z).exp_().mul_((1 - a) * gy)).scatter_add_(1, label, -(1 - a) * gy)
        out["dlogits"] = g.to(s["logits"].dtype)
    return out


PLAIN = {"attn": _plain_attn, "route": _plain_route, "distill": _plain_distill}


def _plain(s):
    with torch.no_grad():
        return PLAIN[s["kind"]](s)


# --------------------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------------------
def _own(s):
    from mlperf_training_b200.ops import functional as F
    from mlperf_training_b200.ops import moe_ops as M
    with torch.set_grad_enabled(s["train"]):
        if s["kind"] == "attn":
            mask = F.attention_mask(s["B"], s["Sq"], s["Skv"], causal=s["causal"], window=s["window"], documents=s["documents"],
                                    prefix=s["flags"] if s["prefix"] else None, device=s["q"].device)
            y = F.masked_attention(s["q"], s["k"], s["v"], mask, softcap=s["softcap"], slopes=s["slopes"])
            out = {"out": y.detach()}
            if s["train"]:
                out["dq"], out["dk"], out["dv"] = torch.autograd.grad(y, [s["q"], s["k"], s["v"]], s["dout"])
        elif s["kind"] == "route":
            idx, w, counts = M.route(s["logits"], s["k"], score=s["score"], bias=s["bias"], groups=s["groups"], top_groups=s["top_groups"],
                                     renormalize=s["renormalize"], scale=SCALE)
            out = {"idx": idx, "w": w.detach(), "counts": counts}
            if s["train"]:
                out["dlogits"], = torch.autograd.grad(w, [s["logits"]], s["gw"])
                if s["bias"] is not None:
                    out["bias"] = M.balance_bias(s["bias"], counts, RATE)
        else:
            loss = F.distill_loss(s["logits"], s["labels"], s["ids"], s["values"], alpha=s["alpha"], temperature=s["temperature"], rest=s["rest"])
            out = {"loss": loss.detach()}
            if s["train"]:
                out["dlogits"], = torch.autograd.grad(loss, [s["logits"]], s["gy"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------
def _pairs(case):
    """How many (query, key) pairs of one head are visible, over all sequences."""
    n, first, w = 0, case["Skv"] - case["Sq"], case["window"]
    for row in _layout(case):
        for s, e, p in row:
            q = torch.arange(max(s, first), e, dtype=torch.int64)
            hi = torch.maximum(q + 1, torch.tensor(p)) if case["causal"] else torch.full_like(q, e)
            lo = torch.clamp(q - w + 1, min=s) if w else torch.full_like(q, s)
            n += int((hi - lo).clamp(min=0).sum())
    return n


def work(case):
    if case["kind"] == "attn":
        B, Sq, Skv, Hq, Hkv, D, t = (case[n] for n in ("B", "Sq", "Skv", "Hq", "Hkv", "D", "train"))
        live = sum(e - s for row in _layout(case) for s, e, _ in row)          # keys that some query may see
        b = 2 * D * (2 * B * Sq * Hq + 2 * live * Hkv) * (2 if t else 1) + (2 * D * B * Sq * Hq if t else 0)
        b += 4 * B * Skv if case["docs"] or case["pad"] else 0
        return {"bytes": b, "flops": (14 if t else 4) * D * Hq * _pairs(case)}
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": T * E * size * (2 if case["train"] else 1) + T * k * (12 if case["train"] else 8) + 4 * E, "flops": T * E * (10 + k)}
    T, V, K = case["T"], case["V"], case["K"]
    size = 2 if case["dtype"] == "bf16" else 4
    both = 2 if case["temperature"] != 1 and case["alpha"] < 1 else 1          # exponentials an element
    return {"bytes": T * V * size * (2 if case["train"] else 1) + T * (K * 12 + 12), "flops": T * V * (4 + 4 * both) * (2 if case["train"] else 1)}


# --------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------
def _exact_attn(s):
    B, Sq, Skv, Hq, Hkv, D = (s[n] for n in ("B", "Sq", "Skv", "Hq", "Hkv", "D"))
    group, first = Hq // Hkv, Skv - Sq
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=DEV)
    grads = {"dq": torch.zeros_like(out), "dk": torch.zeros(B, Skv, Hkv, D, dtype=torch.float64, device=DEV)}
    grads["dv"] = torch.zeros_like(grads["dk"])
    # one document and one key head at a time
    for b, row in enumerate(_layout(s)):
        for lo, hi, pre in row:
            q0 = max(lo, first)
            if q0 >= hi:
                continue
            i, j = torch.arange(q0, hi, device=DEV)[:, None], torch.arange(lo, hi, device=DEV)[None, :]
            see = (j < pre) | (j <= i) if s["causal"] else torch.ones(hi - q0, hi - lo, dtype=torch.bool, device=DEV)
            if s["window"]:
                see = see & (i < j + s["window"])
            for h in range(Hkv):
                heads = slice(h * group, (h + 1) * group)
                q = s["q"][b, q0 - first:hi - first, heads].detach().double().requires_grad_(s["train"])
                k = s["k"][b, lo:hi, h].detach().double().requires_grad_(s["train"])
                v = s["v"][b, lo:hi, h].detach().double().requires_grad_(s["train"])
                x = torch.einsum("ihd,jd->hij", q, k) / D ** 0.5
                if s["softcap"]:
                    x = s["softcap"] * torch.tanh(x / s["softcap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][heads].double()[:, None, None] * (i - j).abs()
                y = torch.einsum("hij,jd->ihd", torch.softmax(torch.where(see, x, -math.inf), -1), v)
                out[b, q0 - first:hi - first, heads] = y.detach()
                if s["train"]:
                    g = torch.autograd.grad(y, [q, k, v], s["dout"][b, q0 - first:hi - first, heads].double())
                    grads["dq"][b, q0 - first:hi - first, heads] = g[0]
                    grads["dk"][b, lo:hi, h], grads["dv"][b, lo:hi, h] = g[1], g[2]
    return {"out": out, **grads} if s["train"] else {"out": out}


def _exact_route(s):
    import numpy as np
    T, E, k, G = s["T"], s["E"], s["k"], s["groups"]
    x = s["logits"].detach().double().requires_grad_(True)
    score = 1 / (1 + torch.exp(-x)) if s["score"] == "sigmoid" else torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
    by = score.detach().cpu().numpy()
    if s["bias"] is not None:
        by = by + s["bias"].double().cpu().numpy()
    if s["top_groups"] < G:
        parts = -np.sort(-by.reshape(T, G, E // G), axis=2)[:, :, :2].sum(2)
        order = np.argsort(-parts, axis=1, kind="stable")
        rank = np.empty_like(order)
        np.put_along_axis(rank, order, np.arange(G)[None, :], 1)
        by = np.where(np.repeat(rank < s["top_groups"], E // G, axis=1), by, -np.inf)
    idx = np.argsort(-by, axis=1, kind="stable")[:, :k].copy()
    w = torch.take_along_dim(score, torch.from_numpy(idx).to(DEV), 1)
    if s["renormalize"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    w = SCALE * w
    out = {"idx": None, "w": w.detach(), "counts": None}
    if s["train"]:
        out["dlogits"], = torch.autograd.grad(w, x, s["gw"].double())
        if s["bias"] is not None:
            n = np.bincount(idx.ravel(), minlength=E)
            step = np.where(n * E < T * k, RATE, np.where(n * E > T * k, -RATE, 0.0))
            out["bias"] = s["bias"].double() + torch.from_numpy(step).to(DEV)
    return out


def _exact_distill(s):
    T, a, tau = s["T"], s["alpha"], s["temperature"]
    loss = torch.zeros(T, dtype=torch.float64, device=DEV)
    grad = torch.zeros(T, s["V"], dtype=torch.float64, device=DEV) if s["train"] else None
    step = max(1, (1 << 27) // s["V"])
    for n in range(0, T, step):
        rows = slice(n, min(T, n + step))
        x = s["logits"][rows].detach().double().requires_grad_(s["train"])
        ids, t, labels = s["ids"][rows], s["values"][rows].double(), s["labels"][rows]
        logq = torch.log_softmax(x / tau, 1)
        logp = t if s["rest"] else torch.log_softmax(t / tau, 1)
        events = logp.exp() * (logp - logq.gather(1, ids))
        kl = events.sum(1)
        if s["rest"]:
            r = torch.clamp(1 - logp.exp().sum(1), min=0)
            outside = torch.ones_like(logq, dtype=torch.bool).scatter_(1, ids, False)
            kl = kl + torch.xlogy(r, r) - r * torch.logsumexp(torch.where(outside, logq, -math.inf), 1)
        y = a * tau ** 2 * kl
        if a < 1:
            y = y + (1 - a) * torch.nn.functional.cross_entropy(x, labels.clamp(min=0), reduction="none")
        y = torch.where(labels == -100, torch.zeros_like(y), y)
        loss[rows] = y.detach()
        if s["train"]:
            grad[rows], = torch.autograd.grad(y, x, s["gy"][rows].double())
    return {"loss": loss, "dlogits": grad} if s["train"] else {"loss": loss}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.set_grad_enabled(case["train"] or case["kind"] == "route"):
        return {"attn": _exact_attn, "route": _exact_route, "distill": _exact_distill}[case["kind"]](s)
