"""Shared builders of the window attention tests (not collected by pytest)."""
from __future__ import annotations

import copy

import torch

from fp4_cases import D, Rows
from oracle import window as owin


class WindowRows(Rows):
    """``Rows`` under a window.  Keys that no query of their row sees become NaN (E4M3FN: NaN codes, 4 bits: NaN scales), and
    pages of such keys leave the table."""

    def __init__(self, fmt, lens, chunks=(), window=100, sinks=4, give_back=True, **over):
        super().__init__(fmt, lens, chunks, **over)
        self.window, self.sinks = window, sinks
        if not give_back:
            return
        for first, n, m, table in self.rows():
            m = max(m, 0)
            used = owin.visible(n, m, m - n, window, sinks).any(0)
            for j in (~used).nonzero()[:, 0].tolist():
                page, off = table[j // self.block], j % self.block
                if not 0 <= page < self.blocks:
                    continue
                for side in (0, 1):
                    x, sc = self.pool.side[side], self.pool.scale[side]
                    if fmt == "bf16":
                        x[page, off] = float("nan")
                    elif fmt == "fp8":
                        x[page, off], sc[page, off] = 0x7F, float("nan")
                    else:
                        sc[page, :, off] = 0xFF
            for b in range(-(-m // self.block)):
                if not used[b * self.block:(b + 1) * self.block].any():
                    table[b] = (-1, 10 ** 6, -7)[b % 3]

    def attend(self):
        """(out, bound of the outputs' error), in 64 bits; the bound is ``Rows.attend``'s."""
        out = torch.zeros(self.tokens, self.hq, D, dtype=torch.float64)
        bound = torch.zeros_like(out)
        for first, n, m, table in self.rows():
            m = max(m, 0)
            k, seen = self.pool.values(table, m, 0)
            v, _ = self.pool.values(table, m, 1)
            o, size, logit = owin.attend(self.q[first:first + n].double(), k, v, m - n, self.scale, self.window, self.sinks, seen)
            out[first:first + n] = o
            spread = size + o.abs()
            fp32 = 2 * (D + 4) * 2.0 ** -24 * logit * abs(self.scale)
            bound[first:first + n] = (2.0 ** -8 * (spread + o.abs()) + fp32[..., None] * spread) * 1.02 + 1e-30
        return out, bound

    def part(self, lens, chunks, tables, queries):
        """Other rows over the same pool: lengths, (queries, prefix), their tables and their queries' rows of ``q``."""
        one = copy.copy(self)
        one.lens, one.chunks, one.tables, one.q = list(lens), list(chunks), list(tables), self.q[queries]
        one.tokens = len(one.lens) + sum(n for n, _ in one.chunks)
        return one
