"""Accumulated attention weights and eviction by them -- CPU definition.

``attend`` is the paged attention of one row in 64 bits, with its weights;
``accumulate`` adds a row's weights to its keys' scores (new keys start from
their own sum); ``evict`` chooses what a row over its budget keeps.  Pages that
are not in the pool count as unseen keys.  The reference has no counterpart.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def attend(q, k, v, prefix, scale, seen=None):
    """q [n, H, D], k / v [m, Hkv, D] fp64; query i sees key j <= prefix + i (and ``seen[j]``).

    Returns (out [n, H, D], weights [n, H, m], sum of w|v| [n, H, D], largest sum of |q k| [n, H])."""
    n, heads, _ = q.shape
    m, hkv, d = k.shape
    group = heads // hkv
    kk = k.repeat_interleave(group, 1).permute(1, 0, 2)
    vv = v.repeat_interleave(group, 1).permute(1, 0, 2)
    s = torch.matmul(q.permute(1, 0, 2), kk.transpose(1, 2)) * scale
    mask = torch.arange(m)[None] <= prefix + torch.arange(n)[:, None]
    if seen is not None:
        mask &= seen[None]
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True) if m else torch.zeros(heads, n, 1, dtype=torch.float64)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    size = torch.matmul(q.abs().permute(1, 0, 2), kk.abs().transpose(1, 2)).amax(-1) if m else torch.zeros(heads, n)
    back = lambda x: x.permute(1, 0, 2).contiguous()  # noqa: E731
    return back(torch.matmul(w, vv)), back(w), back(torch.matmul(w, vv.abs())), size.T


def accumulate(scores, weights, table, new_from, block):
    """Adds ``weights`` [n, H, m] of one row to ``scores`` [blocks, Hkv, block] (fp64) in place."""
    hkv = scores.shape[1]
    n, heads, m = weights.shape
    w = weights.view(n, hkv, heads // hkv, m).sum((0, 2))
    for j in range(m):
        page = table[j // block]
        if 0 <= page < scores.shape[0]:
            old = 0.0 if j >= new_from else scores[page, :, j % block]
            scores[page, :, j % block] = old + w[:, j]


def choose(weights: np.ndarray, budget: int, recent: int) -> list[int]:
    """Kept positions of one (row, kv head), ascending: ``weights`` [n] of its tokens."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    old = n - recent
    key = [(-math.inf if math.isnan(w) else w) for w in weights[:old]]
    nan = [math.isnan(w) for w in weights[:old]]
    heavy = sorted(range(old), key=lambda j: (nan[j], -key[j], j))[:budget - recent]
    return sorted(heavy) + list(range(old, n))
