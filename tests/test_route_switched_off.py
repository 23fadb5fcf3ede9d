"""Infinite biases among groups on the CPU, against the definition token by token."""
import math

import pytest
import torch

from mlperf_training_b200.ops import moe_ops as M
from tests import route_oracle as R

CASES = [(8, 4, 2, 2), (12, 4, 2, 3), (64, 8, 3, 6), (60, 5, 2, 4)]


def switched(T, E, G, kind):
    """Logits, and biases of which some groups have all but one expert off ("off"), one expert on ("on"), or one on and the others off ("both"), which
    leaves them a sum without a value: as -inf."""
    g = torch.Generator().manual_seed(E + G)
    x, bias, n = 1.5 * torch.randn(T, E, generator=g), 0.1 * torch.randn(E, generator=g), E // G
    for i in range(0, G, 2):
        at = slice(i * n, (i + 1) * n)
        if kind != "on":
            bias[at] = -math.inf
        bias[i * n + i % n] = 0.1 if kind == "off" else math.inf
    return x, bias


@pytest.mark.parametrize("score", M.ROUTE_SCORES)
@pytest.mark.parametrize("kind", ["off", "on", "both"])
@pytest.mark.parametrize("E,G,top,k", CASES)
def test_groups_with_infinite_biases(E, G, top, k, kind, score):
    x, bias = switched(50, E, G, kind)
    idx, w, counts = M.route(x, k, score=score, bias=bias, groups=G, top_groups=top)
    n = E // G
    for t, row in enumerate(x.double().tolist()):
        s = R.scores(row, score)
        c = [a + b for a, b in zip(s, bias.tolist())]
        value = [sum(sorted(c[i * n:(i + 1) * n], reverse=True)[:2]) for i in range(G)]
        value = [-math.inf if math.isnan(v) else v for v in value]
        stay = sorted(range(G), key=lambda i: (-value[i], i))[:top]
        pool = [e for i in sorted(stay) for e in range(i * n, (i + 1) * n)]
        assert idx[t].tolist() == sorted(pool, key=lambda e: (-c[e], e))[:k]
    assert torch.equal(counts, torch.bincount(idx.flatten(), minlength=E).int())
