"""Masked attention from its definition in 64 bits: truth values element by element, softmax row by row, gradients by autograd."""
import math

import torch


def visible(B, Sq, Skv, causal=True, window=0, documents=None, prefix=None):
    """[B, Sq, Skv], by walking from the query to the key."""
    out = torch.zeros(B, Sq, Skv, dtype=torch.bool)
    for b in range(B):
        ids = [0] * Skv if documents is None else documents[b].tolist()
        flag = [False] * Skv if prefix is None else prefix[b].tolist()
        start = [0] * Skv
        for i in range(1, Skv):
            start[i] = start[i - 1] if ids[i] == ids[i - 1] else i
        lead = [flag[i] and (start[i] == i or False) for i in range(Skv)]
        for i in range(1, Skv):
            lead[i] = flag[i] and (start[i] == i or lead[i - 1])
        for i in range(Sq):
            p = i + Skv - Sq
            for k in range(Skv):
                if ids[p] < 0 or start[p] != start[k]:
                    continue
                if causal and k > p and not lead[k]:
                    continue
                if window and p - k >= window:
                    continue
                out[b, i, k] = True
    return out


def attention(q, k, v, ok, scale=None, softcap=0.0, slopes=None, sink=None):
    """64-bit output of ``q [B, Sq, Hq, D]``; differentiable."""
    B, Sq, Hq, D = q.shape
    Skv, g = k.shape[1], Hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    rows = []
    dist = (torch.arange(Skv)[None, :] - torch.arange(Skv - Sq, Skv)[:, None]).abs().double()
    for b in range(B):
        heads = []
        for h in range(Hq):
            s = q[b, :, h] @ k[b, :, h // g].t() * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[h].double() * dist
            s = s.masked_fill(~ok[b], -math.inf)
            if sink is not None:
                s = torch.cat([s, sink[h].expand(Sq, 1)], 1)
            live = (s > -math.inf).any(1, keepdim=True)
            p = torch.softmax(torch.where(live, s, 0.0), 1)[:, :Skv]
            heads.append(torch.where(live, p, 0.0) @ v[b, :, h // g])
        rows.append(torch.stack(heads, 1))
    return torch.stack(rows)
