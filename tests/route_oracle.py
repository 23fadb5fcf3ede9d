"""Routing token by token in 64 bits, from the definition alone."""
import math


def scores(x, score):
    if score == "sigmoid":
        return [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in x]
    m = max(x)
    if m == -math.inf:
        return [0.0] * len(x)
    e = [math.exp(v - m) for v in x]
    return [v / sum(e) for v in e]


def route(rows, k, score, bias, groups, top_groups, renormalize, scale):
    """(idx, w, counts) as lists."""
    E = len(rows[0])
    n, idx, w, counts = E // groups, [], [], [0] * E
    for x in rows:
        s = scores(x, score)
        c = [a + b for a, b in zip(s, bias)] if bias is not None else s
        value = [sum(sorted(c[g * n:(g + 1) * n], reverse=True)[:2]) for g in range(groups)]
        stay = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
        pool = [e for g in sorted(stay) for e in range(g * n, (g + 1) * n)]
        by = x if bias is None else c
        pick = sorted(pool, key=lambda e: (-by[e], e))[:k]
        total = sum(s[e] for e in pick) + 1e-20 if renormalize else 1.0
        idx.append(pick)
        w.append([scale * s[e] / total for e in pick])
        for e in pick:
            counts[e] += 1
    return idx, w, counts


def grad(rows, gw, k, score, bias, groups, top_groups, renormalize, scale):
    """dL/dlogits by the chain rule over the chosen experts of each token."""
    idx, _, _ = route(rows, k, score, bias, groups, top_groups, renormalize, scale)
    out = []
    for x, g, pick in zip(rows, gw, idx):
        s = scores(x, score)
        total = sum(s[e] for e in pick) + 1e-20
        ds = {}
        for j, e in enumerate(pick):
            # w_i = scale s_i / total: dw_i / ds_e = scale (delta_ie - s_i / total) / total
            if renormalize:
                ds[e] = sum(g[i] * scale * ((f == e) - s[f] / total) / total for i, f in enumerate(pick))
            else:
                ds[e] = g[j] * scale
        if score == "sigmoid":
            out.append([ds.get(e, 0.0) * s[e] * (1 - s[e]) for e in range(len(x))])
        else:
            r = sum(v * s[e] for e, v in ds.items())
            out.append([s[e] * (ds.get(e, 0.0) - r) for e in range(len(x))])
    return out
