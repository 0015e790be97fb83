"""Attention with a sliding window and visible first tokens -- CPU definition.

The query at position t of a row sees the keys j <= t with j > t - window or
j < sinks.  The reference has no counterpart.
"""
from __future__ import annotations

import math

import torch


def visible(n, m, prefix, window, sinks, seen=None):
    """bool [n, m]: which of m keys the queries at positions prefix, prefix + 1, ... see (``seen[j]``: key j exists)."""
    t, j = prefix + torch.arange(n)[:, None], torch.arange(m)[None]
    mask = (j <= t) & ((j > t - window) | (j < sinks))
    return mask if seen is None else mask & seen[None]


def attend(q, k, v, prefix, scale, window, sinks, seen=None):
    """q [n, H, D], k / v [m, Hkv, D] fp64; a query that sees nothing gives zeros.

    Returns (out [n, H, D], sum of w|v| [n, H, D], largest sum of |q k| over the keys seen [n, H])."""
    n, heads, d = q.shape
    m, hkv, _ = k.shape
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    size, logit = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.float64)
    mask = visible(n, m, prefix, window, sinks, seen)
    for i in range(n):
        at = mask[i].nonzero()[:, 0]
        if not len(at):
            continue
        for h in range(heads):
            kk, vv = k[at, h // (heads // hkv)], v[at, h // (heads // hkv)]
            w = torch.softmax(kk @ q[i, h] * scale, 0)
            out[i, h], size[i, h] = w @ vv, w @ vv.abs()
            logit[i, h] = (kk.abs() @ q[i, h].abs()).max()
    return out, size, logit
