"""Balance loss of the mixture router in 64 bits, written from its definition token by token, with its gradient's formula."""
from __future__ import annotations

import torch


def probs(logits, score_fun):
    x = logits.double()
    if score_fun == 0:
        p = torch.softmax(x, -1)
    else:
        p = torch.softmax(torch.nn.functional.logsigmoid(x), -1)     # the sigmoids themselves end near -745
    return torch.where((x == -float("inf")).all(-1, keepdim=True), torch.zeros_like(p), p)


def balance(logits, ids, score_fun, coef, mask=None, cu=None):
    """(loss, counts, gradient) on the CPU."""
    T, E = logits.shape
    topk = ids.shape[1]
    bounds = [0, T] if cu is None else [int(v) for v in cu]
    B = len(bounds) - 1
    loss, counts, grad = 0.0, torch.zeros(E, dtype=torch.int64), torch.zeros(T, E, dtype=torch.float64)
    for a, z in zip(bounds, bounds[1:]):
        rows = [t for t in range(a, z) if mask is None or bool(mask[t])]
        if not rows:
            continue
        c = torch.zeros(E, dtype=torch.float64)
        for t in rows:
            for e in ids[t].tolist():
                if 0 <= e < E:
                    c[e] += 1
        n = len(rows)
        p = probs(logits[rows], score_fun)
        u = coef * E * c / (B * topk * n * n)
        loss += float((u * p.sum(0)).sum())
        counts += c.long()
        d = p * (u - (p * u).sum(-1, keepdim=True))
        if score_fun == 1:
            d = d * (1 - torch.sigmoid(logits[rows].double()))
        grad[rows] = d
    return loss, counts, grad
