"""Shared builders of the 4-bit pool and score tests (not collected by pytest)."""
from __future__ import annotations

import numpy as np
import torch

from oracle import fp4 as ofp4
from oracle import fp8 as ofp8
from oracle import kv_scores

D = 128
STALE = 0xFF  # scale byte of places that no token was written to: E8M0's NaN


def random_values(g, *shape):
    """bf16 values whose channels differ in size, as keys' do."""
    channel = torch.exp(0.7 * torch.randn(shape[-2], shape[-1], generator=g))
    return (torch.randn(*shape, generator=g) * channel).to(torch.bfloat16)


class Pool:
    """One layer's pool on the CPU in any format, filled with stale bytes and then with tokens."""

    def __init__(self, fmt, blocks, block, hkv, seed=0, d=D):
        g = torch.Generator().manual_seed(seed + 77)
        self.fmt, self.blocks, self.block, self.hkv, self.d = fmt, blocks, block, hkv, d
        if fmt == "bf16":
            self.side = [torch.full((blocks, block, hkv, d), float("nan")).to(torch.bfloat16) for _ in range(2)]
            self.scale = [None, None]
        elif fmt == "fp8":
            self.side = [torch.full((blocks, block, hkv, d), 0x7F, dtype=torch.uint8) for _ in range(2)]
            self.scale = [torch.full((blocks, block, hkv), float("nan")) for _ in range(2)]
        else:
            self.side = [torch.randint(0, 256, (blocks, hkv, block, d // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
            self.scale = [torch.full((blocks, hkv, block, d // 32), STALE, dtype=torch.uint8) for _ in range(2)]
        self.tokens = {}

    def write(self, table, k, v, at=0):
        """Tokens ``k`` / ``v`` [n, hkv, d] bf16 at positions at.. of a row; pages that are not in the pool are left out."""
        for side, x in enumerate((k, v)):
            f = x.float().numpy()
            if self.fmt == "bf16":
                codes, scale = x, None
            elif self.fmt == "fp8":
                codes, scale = ofp8.quantize_kv(f)
            else:
                codes, scale = ofp4.quantize_kv(f)
            for i in range(len(x)):
                page, off = table[(at + i) // self.block], (at + i) % self.block
                if not 0 <= page < self.blocks:
                    continue
                where = (page, slice(None), off) if self.fmt == "fp4" else (page, off)
                self.side[side][where] = codes[i] if scale is None else torch.from_numpy(codes[i])
                if scale is not None:
                    self.scale[side][where] = torch.from_numpy(scale[i])

    def values(self, table, n, side):
        """fp64 [n, hkv, d] of a row's first n tokens (zeros where the page is not in the pool), and which are in it."""
        out = torch.zeros(n, self.hkv, self.d, dtype=torch.float64)
        seen = torch.zeros(n, dtype=torch.bool)
        for b in range(-(-n // self.block)):
            page, lo = table[b], b * self.block
            hi = min(lo + self.block, n)
            if not 0 <= page < self.blocks:
                continue
            seen[lo:hi] = True
            if self.fmt == "bf16":
                x = self.side[side][page].double()
            elif self.fmt == "fp8":
                x = torch.from_numpy(ofp8.decode_array(self.side[side][page].numpy()).astype(np.float64)) * \
                    self.scale[side][page].double()[..., None]
            else:
                x = torch.from_numpy(ofp4.dequantize_kv(self.side[side][page].numpy(), self.scale[side][page].numpy()))
                x = x.transpose(0, 1)
            out[lo:hi] = x[:hi - lo]
        return out, seen

    def device(self, device):
        """(k_cache, v_cache, k_scale, v_scale) as the entry points take them."""
        side = [t.to(device) for t in self.side]
        if self.fmt == "fp4":
            side = [t.view(torch.float4_e2m1fn_x2) for t in side]
        return side[0], side[1], *(None if t is None else t.to(device) for t in self.scale)


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


class Rows:
    """Decode rows of ``lens`` keys and prefill rows (queries, prefix) over one pool."""

    def __init__(self, fmt, lens, chunks=(), hq=32, hkv=8, block=64, seed=0, gain=1.0, scale=D ** -0.5, holes=(),
                 spare=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.chunks, self.hq, self.hkv, self.block, self.scale = list(lens), list(chunks), hq, hkv, block, scale
        totals = self.lens + [max(n + p, 0) for n, p in self.chunks]
        pages = [-(-t // block) for t in totals]
        self.blocks = sum(pages) + 2
        order, at, self.tables = torch.randperm(self.blocks, generator=g).tolist(), 0, []
        width = max(pages + [1]) + spare
        for n in pages:
            self.tables.append(order[at:at + n] + [-1] * (width - n))
            at += n
        for row, page, value in holes:
            self.tables[row][page] = value
        self.pool = Pool(fmt, self.blocks, block, hkv, seed)
        for t, table in zip(totals, self.tables):
            k = random_values(g, t, hkv, D)
            k = (k.float() / k.float().square().mean(-1, keepdim=True).sqrt()).to(torch.bfloat16)
            self.pool.write(table, k, random_values(g, t, hkv, D))
        self.tokens = len(self.lens) + sum(n for n, _ in self.chunks)
        self.q = (gain * torch.randn(self.tokens, hq, D, generator=g)).to(torch.bfloat16)

    def arguments(self, device):
        nd = len(self.lens)
        cu_q, cu_k = [0], [0]
        for n, p in self.chunks:
            cu_q.append(cu_q[-1] + n)
            cu_k.append(cu_k[-1] + n + p)
        a = dict(num_decode=nd, num_prefill=len(self.chunks))
        if nd:
            a.update(decode_lens=i32(self.lens, device), decode_tables=i32(self.tables[:nd], device))
        if self.chunks:
            a.update(prefill_cu_q=i32(cu_q, device), prefill_cu_k=i32(cu_k, device), max_q=max(n for n, _ in self.chunks),
                     max_k=max(n + p for n, p in self.chunks), prefill_tables=i32(self.tables[nd:], device))
        return a

    def rows(self):
        """(first query, queries, keys, table) of each row."""
        at, out = 0, []
        for n, table in zip(self.lens, self.tables):
            out.append((at, 1, n, table))
            at += 1
        for (n, p), table in zip(self.chunks, self.tables[len(self.lens):]):
            out.append((at, n, n + p, table))
            at += n
        return out

    def attend(self):
        """(out, weights of each row, bound of the outputs' error), in 64 bits.

        A weight is rounded to bf16 (2^-8) and divided by the sum of the rounded
        weights, which moves an output by at most 2^-8 sum w|v - out|; the
        output is rounded once (2^-8).  A logit's fp32 sum of 128 products and
        its two scalings move it by at most (128 + 4) 2^-24 sum|q k| scale, a
        weight relatively by that twice (its own and the sum's)."""
        out = torch.zeros(self.tokens, self.hq, D, dtype=torch.float64)
        bound = torch.zeros_like(out)
        weights = []
        for first, n, m, table in self.rows():
            m = max(m, 0)
            k, seen = self.pool.values(table, m, 0)
            v, _ = self.pool.values(table, m, 1)
            o, w, size, logit = kv_scores.attend(self.q[first:first + n].double(), k, v, m - n, self.scale, seen)
            out[first:first + n] = o
            spread = size + o.abs()
            fp32 = 2 * (D + 4) * 2.0 ** -24 * logit * abs(self.scale)
            bound[first:first + n] = (2.0 ** -8 * (spread + o.abs()) + fp32[..., None] * spread) * 1.02 + 1e-30
            weights.append((w, fp32))
        return out, weights, bound
