"""Distillation loss token by token in 64 bits from its definition; the gradient by autograd over it."""
import torch


def token_loss(z, label, ids, values, alpha, tau, rest, ignore=-100):
    """Scalar loss of one token: ``z [V]`` in 64 bits, ``ids`` and ``values`` as lists."""
    V = z.numel()
    if label is not None and label == ignore:
        return (z * 0.0).nan_to_num(0.0, 0.0, 0.0).sum() * 0.0
    q = torch.softmax(z / tau, 0)
    logq = torch.log_softmax(z / tau, 0)
    entries = [(i, t) for i, t in zip(ids, values) if 0 <= i < V and t != float("-inf")]
    kl = torch.zeros((), dtype=torch.float64)
    if entries:
        t = torch.tensor([v for _, v in entries], dtype=torch.float64)
        p = t.exp() if rest else torch.softmax(t / tau, 0)
        for (i, _), pj in zip(entries, p):
            if pj > 0:
                kl = kl + pj * (pj.log() - logq[i])
    else:
        p = torch.zeros(1, dtype=torch.float64)
    if rest:
        r = float(1 - p.sum())
        outside = [v for v in range(V) if v not in {i for i, _ in entries}]
        if r > 0 and outside:
            kl = kl + r * (torch.tensor(r, dtype=torch.float64).log() - q[outside].sum().log())
    loss = alpha * tau ** 2 * kl
    if alpha < 1 and label is not None and 0 <= label < V:
        loss = loss - (1 - alpha) * torch.log_softmax(z, 0)[label]
    return loss


def loss_and_grad(logits, labels, ids, values, gy, **cfg):
    z = logits.double().requires_grad_(True)
    cfg = dict(alpha=cfg.get("alpha", 1.0), tau=cfg.get("temperature", 1.0), rest=cfg.get("rest", False), ignore=cfg.get("ignore_index", -100))
    rows = [token_loss(z[t], None if labels is None else int(labels[t]), ids[t].tolist(), values[t].double().tolist(), **cfg)
            for t in range(z.shape[0])]
    loss = torch.stack(rows)
    (loss * gy.double()).sum().backward()
    return loss.detach(), z.grad
