"""Token sampling in 64 bits, one row at a time: the definition that
``mi_b200.sampling.sample_tokens`` is tested against."""
from __future__ import annotations

import math

import numpy as np


def sample_row(x, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """``(token, log-probability, kept tokens)`` of one row of logits."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if not (x > -np.inf).any():
        return -1, -math.inf, []
    top = x.max()
    with np.errstate(invalid="ignore"):
        d = np.where(x == top, 0.0, x - top)
    logz = math.log(np.exp(d).sum())
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not temperature > 0:
        kept = order[:1]
    else:
        if 0 < top_k < len(x):
            order = order[:top_k]
        w = np.exp(d[order] / temperature)
        if top_p < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            keep = before < top_p * w.sum()
            keep[0] = True
            order, w = order[keep], w[keep]
        if min_p > 0:
            order = order[w >= min(min_p, 1.0)]
        kept = np.sort(order)
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    c = np.cumsum(np.exp(d[kept] / temperature) if temperature > 0 else np.ones(1))
    token = int(kept[np.searchsorted(c, u * c[-1], side="right")])
    return token, float(d[token] - logz), kept.tolist()
