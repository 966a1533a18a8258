"""Accumulated attention weights and eviction by them, in 64 bits and one
request at a time: the definitions the kernels are tested against."""
from __future__ import annotations

import numpy as np


def request_tokens(indptr, indices, last, b, page_size):
    """Pages and token count of request ``b`` of a CSR page table."""
    pages = np.asarray(indices[indptr[b]:indptr[b + 1]], np.int64)
    n = (len(pages) - 1) * page_size + int(last[b]) if len(pages) else 0
    return pages, n


def decode_weights(q, k, scale):
    """``q [Hq, D]``, ``k [n, Hkv, D]`` -> weights ``[n, Hkv]`` summed over groups."""
    hq, d = q.shape
    n, hkv, _ = k.shape
    z = np.einsum("hgd,nhd->hgn", np.asarray(q, np.float64).reshape(hkv, hq // hkv, d),
                  np.asarray(k, np.float64)) * scale
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).sum(1).T


def prompt_weights(q, k, scale, window=0, causal=True, lse=None):
    """``q [nq, Hq, D]``, ``k [n, Hkv, D]`` -> ``[n, Hkv]``: weights given by the
    last ``window`` queries (0: all), bottom-right causal. ``lse [nq, Hq]``:
    the rows' log-sum-exp (default: computed)."""
    nq, hq, d = q.shape
    n, hkv, _ = k.shape
    out = np.zeros((n, hkv))
    first = max(0, nq - window) if window else 0
    qd, kd = np.asarray(q, np.float64), np.asarray(k, np.float64)
    for h in range(hq):
        z = qd[first:, h] @ kd[:, h // (hq // hkv)].T * scale
        if causal:
            seen = np.arange(n)[None] <= (n - nq + np.arange(first, nq))[:, None]
            z = np.where(seen, z, -np.inf)
        if lse is None:
            m = z.max(-1, keepdims=True, initial=-np.inf)
            m = np.where(np.isfinite(m), m, 0.0)
            s = np.exp(z - m).sum(-1, keepdims=True)
            w = np.where(s > 0, np.exp(z - m) / np.where(s > 0, s, 1.0), 0.0)
        else:
            row = np.asarray(lse, np.float64)[first:, h, None]
            w = np.where(np.isfinite(row), np.exp(z - np.where(np.isfinite(row), row, 0.0)), 0.0)
        out[:, h // (hq // hkv)] += w.sum(0)
    return out


def evict_slots(scores, budget, recent, sinks):
    """Source slot of each slot after cutting a head's ``scores [n]`` to ``budget``."""
    s = np.asarray(scores, np.float64)
    n = len(s)
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    low, end = budget - recent, n - recent
    middle = list(range(sinks, end))
    rank = sorted(middle, key=lambda t: (not np.isnan(s[t]), s[t] if not np.isnan(s[t]) else 0.0, -t),
                  reverse=True)
    kept = set(rank[:low - sinks])
    movers = [t for t in range(low, end) if t in kept]
    src = []
    for t in range(low):
        src.append(t if t < sinks or t in kept else movers.pop(0))
    assert not movers
    return src + list(range(end, n))


def evict(kv, scores, indptr, indices, last, budget, recent=0, sinks=0):
    """``kv [P, 2, ps, H, D]`` and ``scores [P, H, ps]`` cut in place; ``kept [B, H, budget]``."""
    ps, heads = kv.shape[2], kv.shape[3]
    kept = np.full((len(last), heads, budget), -1, np.int32)
    for b in range(len(last)):
        pages, n = request_tokens(indptr, indices, last, b, ps)
        for h in range(heads):
            flat = scores[pages, h].reshape(-1)
            src = evict_slots(flat[:n], budget, recent, sinks)
            kept[b, h] = src
            if n <= budget:
                continue
            rows = kv[pages, :, :, h].transpose(0, 2, 1, 3).reshape(len(pages) * ps, 2, -1).copy()
            rows[:budget] = rows[src]
            kv[pages, :, :, h] = rows.reshape(len(pages), ps, 2, -1).transpose(0, 2, 1, 3)
            new = np.zeros_like(flat)
            new[:budget] = flat[src]
            scores[pages, h] = new.reshape(len(pages), ps)
    return kept
