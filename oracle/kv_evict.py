"""Attention weights per cached token and eviction in 64 bits (oracle; see oracle/__init__.py)."""
from __future__ import annotations

import math

import torch


def token_weights(q, k, table, lens, lse, sm_scale, soft_cap=0.0, length=None):
    """sum over the heads of a group of exp(logit - lse): q [B, Hq, D], k [pages, P, Hkv, D] float64, lse [B, Hq].  Returns
    (w [B, Hkv, S], largest [B, Hkv, S]: the largest |logit| + |lse| that went into it)."""
    b, hq, _ = q.shape
    page, hkv = k.shape[1], k.shape[2]
    length = length or max(max(lens), 1)
    w = torch.zeros(b, hkv, length, dtype=torch.float64)
    big = torch.zeros_like(w)
    for i, n in enumerate(lens):
        n = min(n, length)
        if n <= 0:
            continue
        pos = torch.arange(n)
        ki = k[table[i].cpu().long()[pos // page], pos % page]
        s = torch.einsum("hgd,nhd->hgn", q[i].cpu().double().unflatten(0, (hkv, -1)), ki) * sm_scale
        if soft_cap:
            s = soft_cap * torch.tanh(s / soft_cap)
        l = lse[i].cpu().double().unflatten(0, (hkv, -1))[..., None]
        w[i, :, :n] = torch.exp(s - l).sum(1)
        big[i, :, :n] = (s.abs() + l.abs()).amax(1)
    return w, big


def survivors(weights, n: int, keep: int, recent: int):
    """Slots that stay of one head's n tokens, ascending: a list.  Python's sort: by weight, then by slot."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    w = [float(x) for x in weights[:old]]
    rank = sorted(range(old), key=lambda i: (-math.inf if math.isnan(w[i]) else -w[i], 0 if math.isnan(w[i]) else 1, i))
    return sorted(rank[:keep - recent]) + list(range(old, n))


def evict(rows, table, lens, weights, keep: int, recent: int):
    """Apply to CPU tensors: ``rows`` [pages, P, Hkv, ...] tensors, returned moved.  Returns (rows, lens, kept, weights)."""
    rows = [r.clone() for r in rows]
    page, hkv = rows[0].shape[1], rows[0].shape[2]
    kept = torch.full((len(lens), hkv, keep), -1, dtype=torch.int32)
    out = torch.zeros_like(weights)
    for b, n in enumerate(lens):
        n = max(min(n, weights.shape[2], table.shape[1] * page), 0)
        for h in range(hkv):
            stay = survivors(weights[b, h], n, keep, recent)
            kept[b, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            out[b, h, :len(stay)] = weights[b, h, stay]
            for r in rows:
                whole = [r[int(table[b, s // page]), s % page, h].clone() for s in stay]
                for j, x in enumerate(whole):
                    r[int(table[b, j // page]), j % page, h] = x
    new = torch.tensor([min(max(min(n, weights.shape[2], table.shape[1] * page), 0), keep) for n in lens], dtype=torch.int32)
    return rows, new, kept, out
