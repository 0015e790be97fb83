"""The operators of a compressed KV cache, as measurable cases.

A serving engine that runs out of KV pool before it runs out of compute holds
its cache in 4 bits, and drops the tokens that attention no longer looks at:

* ``write``   new K/V rows into a 4-bit pool (``store_kvcache``), and the same
  tokens read back (``load_kvcache``), as a block swap or a format change does.
* ``attend``  ``paged_attention`` over a 4-bit pool: decode rows, chunks of
  prompts, and both.
* ``weigh``   ``accumulate_attention``: the attention weight that a step's
  queries give every cached token, added to the pool's fp32 scores.
* ``evict``   ``evict_kv``: rows over their budget keep the newest and the
  heaviest tokens of every kv head, moved to the front of their pages.

The 4-bit pool holds E2M1 codes, two to a byte (the even channel in the low
half), with one E8M0 scale per 32 channels; its pages are stored head by head,
``[blocks, kv_heads, block_size, ...]``, as the scores' pages are.  bf16 and
E4M3FN pools are ``[blocks, block_size, kv_heads, ...]``.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

HD = 128
SCALE = HD ** -0.5
GROUP = 32             # channels per E8M0 scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOW, HIGH = 63, 252    # scale codes: 2^-64 (the pools' smallest scale) to 2^125 (6 * 2^125 is still finite)


# ------------------------------------------------------------------- cases
def _attn(kind, name=None, rows=0, lo=1, hi=1, plan=0, prefill="", hq=32, hkv=8, kv="fp4", block=256, gain=1.0):
    case = dict(kind=kind, rows=rows, lo=lo, hi=hi, plan=plan, prefill=prefill, hq=hq, hkv=hkv, kv=kv, block=block,
                gain=gain)
    if name:
        case["name"] = name
    return case


def _evict(name=None, rows=1, lo=1, hi=1, plan=0, budget=1, recent=0, hkv=8, kv="bf16", block=256, layers=1):
    case = dict(kind="evict", rows=rows, lo=lo, hi=hi, plan=plan, budget=budget, recent=recent, hkv=hkv, kv=kv,
                block=block, layers=layers)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # The new tokens of a decode step of 24 sequences.
        dict(kind="write", name="write_24", tokens=24, hkv=8, block=256),
        # A prompt's tokens, or 16 blocks swapped in.
        dict(kind="write", name="write_4096", tokens=4096, hkv=8, block=256),
        # One user's tokens one at a time: the smallest step there is.
        _attn("attend", "attend_1row", 1, 300, 1000, plan=1),
        # A loaded server: 64 long conversations.
        _attn("attend", "attend_64rows", 64, 512, 4096, plan=3),
        # A few very long documents, which a 4-bit pool is for.
        _attn("attend", "attend_long", 3, 20000, 60000, plan=5, gain=2.0),
        # The mixed step of the chunked scheduler: decode rows first, then two chunks.
        _attn("attend", "attend_24d_2x512", 24, 256, 4096, plan=5, prefill="512:0,512:1024"),
        # Ragged chunks of prompts without decode rows, on one of two tensor-parallel ranks.
        _attn("attend", "attend_chunks", prefill="1000:2500,300:700,77:3000", hq=16, hkv=4, gain=2.0),
        # The weights of a lightly loaded decode step, pool not quantised.
        _attn("weigh", "weigh_16rows", 16, 64, 1024, plan=2, kv="bf16", gain=3.0),
        # The weights of a loaded decode step on a 4-bit pool.
        _attn("weigh", "weigh_64rows_fp4", 64, 512, 4096, plan=3, gain=3.0),
        # The weights of two prompts' chunks on an E4M3FN pool.
        _attn("weigh", "weigh_chunks_fp8", prefill="1024:1024,500:0", kv="fp8", gain=3.0),
        # One conversation over its budget, one layer.
        _evict("evict_1row", 1, 1500, 1500, plan=1, budget=1024, recent=128),
        # A batch of long conversations cut back to a quarter, eight layers of a 4-bit pool in one call.
        _evict("evict_8layers_fp4", 16, 3000, 8192, plan=2, budget=2048, recent=256, kv="fp4", layers=8),
    ]


_HEADS = ((32, 8), (32, 8), (16, 4), (28, 4), (40, 8), (8, 8), (16, 2), (64, 8), (16, 1))


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("write", "attend", "attend", "attend", "weigh", "weigh", "evict"))
    hq, hkv = rng.choice(_HEADS)
    plan = rng.randrange(1 << 20)
    block = rng.choice((64, 128, 192, 256, 256, 512))
    if kind == "write":
        return dict(kind="write", tokens=log(1, 4096), hkv=hkv, block=block)
    if kind == "evict":
        kv = rng.choice(("bf16", "fp8", "fp4"))
        layers = rng.choice((1, 2, 4, 8))
        hi = log(80, 16384)
        budget = max(2, int(hi * rng.uniform(0.1, 0.9)))
        # No more bytes moved than by the largest listed one.
        most = 300_000_000 // (layers * hkv * (8 * hi + 4 * budget * _ROW[kv]))
        return _evict(None, max(1, min(log(1, 64), most)), max(1, hi // 4), hi, plan, budget, rng.randrange(budget + 1),
                      hkv, kv, block, layers)
    kv = "fp4" if kind == "attend" else rng.choice(("bf16", "fp8", "fp4"))
    gain = rng.choice((1.0, 2.0, 3.0))
    what = rng.choice(("decode", "decode", "prefill", "mixed"))
    rows, hi, chunks = 0, 1, []
    if what != "prefill":
        hi = log(16, 60000 if what == "decode" else 4096)
        rows = max(1, min(log(1, 64), 150_000 // hi))
    if what != "decode":
        # Together no more (query, key) pairs than the largest listed chunks.
        room = (2_000_000 if what == "prefill" else 1_000_000) * 16 // max(16, hq)
        for _ in range(rng.randint(1, 3)):
            n, prefix = log(1, 1024), rng.choice((0, log(1, 4096)))
            while n * prefix + n * (n + 1) // 2 > room and n > 1:
                n //= 2
            room -= n * prefix + n * (n + 1) // 2
            chunks.append("%d:%d" % (n, prefix))
            if room < 50_000:
                break
    return _attn(kind, None, rows, max(1, hi // 8), hi, plan, ",".join(chunks), hq, hkv, kv, block, gain)


def _chunks(case):
    return [tuple(int(x) for x in c.split(":")) for c in case["prefill"].split(",")] if case["prefill"] else []


def _lens(case):
    """Key counts of the decode rows: the same for every seed, as they set the work."""
    rng = random.Random(case["plan"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["rows"])]


_ROW = {"bf16": 2 * HD, "fp8": HD + 4, "fp4": HD // 2 + HD // GROUP}  # bytes of one key (or value) of one kv head


def work(case):
    hkv = case["hkv"]
    if case["kind"] == "write":
        n = case["tokens"] * hkv * 2
        return {"bytes": n * 2 * (2 * HD + _ROW["fp4"]) + 8 * case["tokens"], "flops": 0}
    row = _ROW[case["kv"]]
    if case["kind"] == "evict":
        # Scores of every token read; rows over budget: kept rows moved, their scores written, the rest cleared.
        total = 0
        for n in _lens(case):
            over = n > case["budget"]
            total += 4 * n + (4 * case["budget"] * row + 4 * n if over else 0) + 4 * min(n, case["budget"])
        return {"bytes": total * case["layers"] * hkv, "flops": 0}
    keys = sum(_lens(case)) + sum(n + p for n, p in _chunks(case))
    pairs = sum(_lens(case)) + sum(n * p + n * (n + 1) // 2 for n, p in _chunks(case))
    queries = case["rows"] + sum(n for n, _ in _chunks(case))
    if case["kind"] == "attend":
        return {"bytes": keys * hkv * 2 * row + queries * case["hq"] * HD * 4, "flops": 4 * HD * case["hq"] * pairs}
    return {"bytes": keys * hkv * (row + 8) + queries * case["hq"] * HD * 2, "flops": 2 * HD * case["hq"] * pairs}


# ------------------------------------------------------- the formats, plainly
def _fp4_encode(x):
    """bf16 ``[..., D]`` -> packed codes uint8 ``[..., D/2]`` and scale codes uint8 ``[..., D/32]``.

    The scale is the smallest power of two at which the largest magnitude of
    its 32 channels is below 7 (7 is where rounding would leave 6); codes are
    the nearest E2M1 value, ties to the even code, saturating at 6.
    """
    bits = x.contiguous().view(torch.int16).int()
    sign, mag = (bits >> 15) & 1, bits & 0x7FFF
    mag = mag.clamp(max=0x7F7F)  # infinities and NaN count as the largest finite value
    mag = mag.view(*mag.shape[:-1], -1, GROUP)
    scale = (((mag.amax(-1) + 32) >> 7) - 2).clamp(LOW, HIGH)
    y = torch.ldexp(mag.short().view(torch.bfloat16).float(), (127 - scale)[..., None])
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
            + (y >= 3.5).int() + (y > 5.0).int())
    code = code.view(x.shape) + 8 * sign
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def _fp4_decode(packed, scale):
    """fp32 values ``[..., D]`` of packed codes ``[..., D/2]`` and scale codes ``[..., D/32]``."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)
    v = table[code.int()].view(*scale.shape, GROUP)
    return torch.ldexp(v, scale.int()[..., None] - 127).view(code.shape)


def _fp8_encode(x):
    xf = x.float()
    amax = xf.abs().amax(-1, keepdim=True)
    scale = torch.where(amax == 0, torch.ones_like(amax), (amax / 448.0).clamp(min=2.0 ** -64))
    return (xf / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale[..., 0].contiguous()


def _values(pages, scale, kv):
    """fp32 ``[..., block, kv_heads, D]`` of pool pages."""
    if kv == "bf16":
        return pages.float()
    if kv == "fp8":
        return pages.view(torch.float8_e4m3fn).float() * scale[..., None]
    return _fp4_decode(pages, scale).transpose(-2, -3)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _unit(x):
    return x / x.square().mean(-1, keepdim=True).sqrt()


def _pool(g, blocks, block, hkv, kv, key):
    """One side of a pool filled with tokens' K (unit RMS, a few strong channels) or V, and its scales."""
    channel = torch.exp(0.5 * _randn(g, hkv, HD))
    pages, scales = [], []
    for at in range(0, blocks, 512):
        x = _randn(g, min(512, blocks - at), block, hkv, HD)
        x = (_unit(x * channel) if key else x).to(torch.bfloat16)
        if kv == "bf16":
            pages.append(x)
        else:
            c, s = _fp8_encode(x) if kv == "fp8" else _fp4_encode(x.transpose(1, 2))
            pages.append(c.contiguous())
            scales.append(s.contiguous())
    return torch.cat(pages), torch.cat(scales) if scales else None


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(pages, seed):
    """Block tables of rows of so many pages, -1 padded, and the pool's block count."""
    order = list(range(sum(pages) + 2))
    random.Random(seed).shuffle(order)
    width, rows, at = max(pages), [], 0
    for n in pages:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return _i32(rows), len(order)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    block, hkv = case["block"], case["hkv"]
    up = lambda n: -(-n // block)  # noqa: E731
    if case["kind"] == "write":
        n = case["tokens"]
        blocks = up(n) + 2
        qkv = _randn(g, n, (32 + 2 * hkv) * HD).to(torch.bfloat16)  # K and V are views of the fused projection's output
        slots = torch.randperm(blocks * block, generator=g, device="cuda")[:n].int() if n <= 256 else \
            torch.arange(n, device="cuda", dtype=torch.int32) + block
        pool = [torch.zeros(blocks, hkv, block, w, dtype=torch.uint8, device="cuda")
                for w in (HD // 2, HD // 2, HD // GROUP, HD // GROUP)]
        kv = qkv[:, 32 * HD:].view(n, 2 * hkv, HD)
        return dict(case=case, k=kv[:, :hkv], v=kv[:, hkv:], slots=slots, kc=pool[0], vc=pool[1], ks=pool[2], vs=pool[3])
    lens = _lens(case)
    if case["kind"] == "evict":
        tables, blocks = _tables([up(n) for n in lens], seed)
        layers = case["layers"]
        sides = [_pool(g, layers * blocks, block, hkv, case["kv"], key) for key in (True, False)]
        (kc, ks), (vc, vs) = [tuple(None if t is None else t.view(layers, blocks, *t.shape[1:]) for t in s) for s in sides]
        # Accumulated weights: heavy-tailed, some tokens never looked at and so equal.
        scores = torch.exp(2.0 * _randn(g, layers, blocks, hkv, block)) * (_randn(g, layers, blocks, hkv, block) > -1.0)
        keep = torch.arange(case["budget"], device="cuda")
        page = tables.long().clamp(min=0)[:, (keep // block).clamp(max=tables.shape[1] - 1)]
        slots = torch.where(keep[None] < _i32(lens)[:, None], page * block + keep % block, -1)
        slots = torch.where(slots[None] < 0, -1, slots[None] + torch.arange(layers, device="cuda").view(-1, 1, 1) * blocks * block)
        return dict(case=case, kc=kc, vc=vc, ks=ks, vs=vs, scores=scores, live=scores.clone(), lens=_i32(lens),
                    tables=tables, slots=slots.reshape(-1).int())
    chunks = _chunks(case)
    all_tables, blocks = _tables([up(n) for n in lens] + [up(n + p) for n, p in chunks], seed)
    tokens = len(lens) + sum(n for n, _ in chunks)
    q = (case["gain"] * _unit(_randn(g, tokens, case["hq"], HD))).to(torch.bfloat16)
    kc, ks = _pool(g, blocks, block, hkv, case["kv"], True)
    vc, vs = _pool(g, blocks, block, hkv, case["kv"], False) if case["kind"] == "attend" else (None, None)
    cu_q, cu_k = [0], [0]
    for n, p in chunks:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + n + p)
    nd = len(lens)
    rows = dict(num_decode=nd, decode_lens=_i32(lens) if nd else None, decode_tables=all_tables[:nd].contiguous() if nd else None,
                num_prefill=len(chunks), prefill_cu_q=_i32(cu_q) if chunks else None,
                prefill_cu_k=_i32(cu_k) if chunks else None, max_q=max([n for n, _ in chunks], default=0),
                max_k=max([n + p for n, p in chunks], default=0),
                prefill_tables=all_tables[nd:].contiguous() if chunks else None)
    scores = _randn(g, blocks, hkv, block).abs() if case["kind"] == "weigh" else None
    return dict(case=case, q=q, kc=kc, vc=vc, ks=ks, vs=vs, rows=rows, scores=scores)


# ---------------------------------------------------------- the plain forms
def _plain_write(s):
    hkv, block = s["kc"].shape[1], s["kc"].shape[2]
    out = []
    page, at = (s["slots"] // block).long(), (s["slots"] % block).long()
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        c, e = _fp4_encode(x)
        codes[page, :, at] = c
        scales[page, :, at] = e
        out.append(_fp4_decode(codes[page, :, at], scales[page, :, at]).to(torch.bfloat16).view(-1, hkv, HD))
    return out


def _gather(s, side, tables):
    """fp32 ``[rows, kv_heads, capacity, D]`` keys or values of the rows' pages."""
    pages, scale = s[side + "c"], s[side + "s"]
    index = tables.long().clamp(min=0)
    x = _values(pages[index], None if scale is None else scale[index], s["case"]["kv"])
    return x.flatten(1, 2).transpose(1, 2)


def _probabilities(s, q, keys, seen):
    """fp32 softmax weights ``[rows, kv_heads, queries * group, capacity]``; ``seen`` masks ``[rows, queries, capacity]``."""
    rows, n, hq, d = q.shape
    hkv = keys.shape[1]
    x = q.float().view(rows, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(rows, hkv, -1, d)
    logits = torch.matmul(x, keys.transpose(-1, -2)) * SCALE
    mask = seen[:, None, :, None].expand(rows, 1, n, hq // hkv, seen.shape[-1]).flatten(2, 3)
    logits = logits.masked_fill(~mask, -math.inf)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _heads_back(o, n, hkv):
    """``[rows, kv_heads, queries * group, D]`` -> bf16 ``[rows, queries, heads, D]``."""
    rows, _, m, d = o.shape
    return o.view(rows, hkv, n, m // n, d).permute(0, 2, 1, 3, 4).reshape(rows, n, -1, d).to(torch.bfloat16)


def _phases(s):
    """(queries ``[rows, n, heads, D]``, tables, key counts, masks, way back to tokens) of the decode rows and of the prompts."""
    r, q, nd = s["rows"], s["q"], s["rows"]["num_decode"]
    block, found = s["case"]["block"], []
    if nd:
        at = torch.arange(r["decode_tables"].shape[1] * block, device=q.device)
        found.append((q[:nd, None], r["decode_tables"], r["decode_lens"], torch.ones_like(r["decode_lens"]),
                      at[None, None] < r["decode_lens"][:, None, None], None))
    if r["num_prefill"]:
        cq = r["prefill_cu_q"].long()
        lq, lk = cq[1:] - cq[:-1], (r["prefill_cu_k"][1:] - r["prefill_cu_k"][:-1]).long()
        token = torch.arange(q.shape[0] - nd, device=q.device)
        row = torch.searchsorted(cq[1:].contiguous(), token, right=True)
        i = token - cq[row]
        padded = torch.zeros(r["num_prefill"], r["max_q"], *q.shape[1:], dtype=q.dtype, device=q.device)
        padded[row, i] = q[nd:]
        at = torch.arange(r["prefill_tables"].shape[1] * block, device=q.device)
        place = torch.arange(r["max_q"], device=q.device)
        seen = (at[None, None] <= place[None, :, None] + (lk - lq)[:, None, None]) & (place[None, :, None] < lq[:, None, None])
        found.append((padded, r["prefill_tables"], lk, lq, seen, (row, i)))
    return found


def _attend_phase(s, q, tables, seen, back):
    o = torch.matmul(_probabilities(s, q, _gather(s, "k", tables), seen), _gather(s, "v", tables))
    o = _heads_back(o, q.shape[1], s["case"]["hkv"])
    return o[:, 0] if back is None else o[back]


def _plain_attend(s):
    return torch.cat([_attend_phase(s, q, tables, seen, back) for q, tables, _, _, seen, back in _phases(s)])


def _weigh_phase(s, scores, q, tables, lk, lq, seen):
    """``scores`` ``[blocks + 1, kv_heads, block]`` (the last for places that are none) with one phase's weights."""
    block, hkv = s["case"]["block"], s["case"]["hkv"]
    w = _probabilities(s, q, _gather(s, "k", tables), seen).sum(2)
    at = torch.arange(w.shape[-1], device=w.device)
    page = torch.where(at[None] < lk[:, None], tables.long()[:, at // block], scores.shape[0] - 1)
    index = (page[:, None], torch.arange(hkv, device=w.device)[None, :, None], (at % block)[None, None])
    new = (at[None] >= (lk - lq)[:, None]) & (at[None] < lk[:, None])
    old = scores[index]
    scores.index_put_(index, torch.where(new[:, None], w, w + old))
    return scores


def _plain_weigh(s):
    scores = torch.cat((s["scores"], torch.zeros_like(s["scores"][:1])))
    [_weigh_phase(s, scores, q, tables, lk, lq, seen) for q, tables, lk, lq, seen, _ in _phases(s)]
    return s["scores"].copy_(scores[:-1])


def _plain_evict(s):
    c, lens, tables = s["case"], s["lens"].long(), s["tables"].long()
    block, budget, recent, hkv, layers = c["block"], c["budget"], c["recent"], c["hkv"], c["layers"]
    live = s["live"].copy_(s["scores"])
    dev = lens.device
    at = torch.arange(tables.shape[1] * block, device=dev)
    layer = torch.arange(layers, device=dev).view(-1, 1, 1, 1)
    head = torch.arange(hkv, device=dev).view(1, 1, -1, 1)
    page = tables.clamp(min=0)[:, at // block][None, :, None]
    weight = live[layer, page, head, at % block]                      # [layers, rows, kv_heads, capacity]
    newest = lens - torch.minimum(lens, torch.full_like(lens, recent))
    order = torch.where(at < newest.view(1, -1, 1, 1), weight, -math.inf)
    place = torch.sort(order, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(place).scatter_(-1, place, at.expand_as(place).contiguous())
    over = (lens > budget).view(1, -1, 1, 1)
    keep = torch.where(over, (rank < budget - recent) | (at >= newest.view(1, -1, 1, 1)), True) & (at < lens.view(1, -1, 1, 1))
    kept = torch.sort(torch.where(keep, at, 1 << 30), dim=-1).values[..., :budget]
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=1 << 30)
    none = kept == 1 << 30
    to = torch.where(none, 0, torch.arange(budget, device=dev))
    kept = torch.where(none, kept[..., :1], kept)                     # places past the row repeat its first token
    rows = torch.arange(len(lens), device=dev).view(1, -1, 1, 1)
    src = (layer, tables[rows, kept // block], kept % block, head)
    dst = (layer, tables[rows, to // block], to % block, head)
    for pool in (s["kc"], s["vc"], s["ks"], s["vs"]):
        if pool is not None:
            pool = pool.transpose(2, 3) if c["kv"] == "fp4" else pool
            pool[dst] = pool[src]
    moved = live[src[0], src[1], src[3], src[2]]
    cleared = torch.where(over & (at < lens.view(1, -1, 1, 1)), 0.0, weight)
    dead = torch.where(at < lens.view(1, -1, 1, 1), at, 0)            # places past the row repeat its first token
    first = torch.where(at < lens.view(1, -1, 1, 1), cleared, cleared[..., :1])
    live[layer, tables[rows, dead // block], head, dead % block] = first
    live[dst[0], dst[1], dst[3], dst[2]] = moved
    return torch.minimum(lens, torch.full_like(lens, budget)).int(), torch.where(none, -1, kept).int(), live


def _plain_rows(s):
    """The kept tokens' K and V of a quantised pool as bf16 ``[tokens, kv_heads, D]``, zeros where there is none."""
    block, kv, out = s["case"]["block"], s["case"]["kv"], []
    slot = s["slots"].long().clamp(min=0)
    for pages, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        pages, scales = pages.flatten(0, 1), scales.flatten(0, 1)
        if kv == "fp8":
            x = pages.flatten(0, 1)[slot].view(torch.float8_e4m3fn).float() * scales.flatten(0, 1)[slot][..., None]
        else:
            x = _fp4_decode(pages[slot // block, :, slot % block], scales[slot // block, :, slot % block])
        out.append(torch.where((s["slots"] >= 0)[:, None, None], x, 0.0).to(torch.bfloat16))
    return out


# --------------------------------------------------------- the framework's
def _framework():
    package = os.path.join(os.getcwd(), "slo-aware-llm-serving-engine_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import slo_attn
    return slo_attn


def _typed(t, kv):
    return t.view(torch.float4_e2m1fn_x2) if kv == "fp4" else t


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        if kind == "write":
            return _plain_write(s)
        if kind == "attend":
            return _plain_attend(s)
        if kind == "weigh":
            return _plain_weigh(s)
        out = _plain_evict(s)
        return (*out, s["kc"], s["vc"]) if c["kv"] == "bf16" else (*out, *_plain_rows(s))
    slo_attn = _framework()
    if kind == "write":
        kc, vc = _typed(s["kc"], "fp4"), _typed(s["vc"], "fp4")
        slo_attn.store_kvcache(s["k"], s["v"], kc, vc, s["slots"], s["ks"], s["vs"])
        return list(slo_attn.load_kvcache(kc, vc, s["slots"], s["ks"], s["vs"]))
    kc = _typed(s["kc"], c["kv"])
    if kind == "attend":
        return slo_attn.paged_attention(s["q"], kc, _typed(s["vc"], "fp4"), SCALE, num_kv_heads=c["hkv"], k_scale=s["ks"],
                                        v_scale=s["vs"], **s["rows"])
    if kind == "weigh":
        slo_attn.accumulate_attention(s["q"], kc, s["scores"], SCALE, num_kv_heads=c["hkv"], k_scale=s["ks"], **s["rows"])
        return s["scores"]
    vc = _typed(s["vc"], c["kv"])
    live = s["live"].copy_(s["scores"])  # the weights of this pass; eviction moves and clears them
    lens, kept = slo_attn.evict_kv(kc, vc, live, s["lens"], s["tables"], c["budget"], c["recent"], s["ks"], s["vs"])
    if c["kv"] == "bf16":
        return lens, kept, live, s["kc"], s["vc"]
    flat = [_typed(t.flatten(0, 1), c["kv"]) for t in (s["kc"], s["vc"])]
    return lens, kept, live, *slo_attn.load_kvcache(*flat, s["slots"], s["ks"].flatten(0, 1), s["vs"].flatten(0, 1))


# ------------------------------------------------------ the definition, in 64 bits
def _nearest(x):
    """The values that 4 bits hold for bf16 rows ``[n, heads, D]``, by distance to all sixteen."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    y = x.double().view(*x.shape[:-1], -1, GROUP)
    top = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7.0))
    e = e + (top >= 7.0 * torch.exp2(e)).double()   # below 7, not at it
    e = torch.where(top == 0, -64.0, e).clamp(LOW - 127, HIGH - 127)
    m = (y / torch.exp2(e)).abs()
    d = (m[..., None] - grid).abs() + 1e-9 * (torch.arange(8, device=x.device) % 2)  # ties to the even code
    return (torch.copysign(grid[d.argmin(-1)], y) * torch.exp2(e)).view(x.shape)


def _double_rows(s, side, table, n):
    """fp64 ``[n, kv_heads, D]`` of a row's first n tokens."""
    block, kv = s["case"]["block"], s["case"]["kv"]
    pages = table[:-(-n // block)].long()
    x = s[side + "c"][pages]
    if kv == "fp4":
        scale = torch.exp2(s[side + "s"][pages].double() - 127)
        lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=x.device)
        v = torch.empty(*x.shape[:-1], HD, dtype=torch.float64, device=x.device)
        v[..., 0::2], v[..., 1::2] = lut[(x % 16).long()], lut[(x // 16).long()]
        x = (v * scale.repeat_interleave(GROUP, -1)).permute(0, 2, 1, 3)
    elif kv == "fp8":
        x = x.view(torch.float8_e4m3fn).double() * s[side + "s"][pages].double()[..., None]
    else:
        x = x.double()
    return x.flatten(0, 1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return [_nearest(s["k"]), _nearest(s["v"])]
    if case["kind"] == "evict":
        return _exact_evict(s)
    r, nd, hkv = s["rows"], s["rows"]["num_decode"], case["hkv"]
    lens, chunks = _lens(case), _chunks(case)
    todo = [(i, 1, n, r["decode_tables"][i]) for i, n in enumerate(lens)]
    at = nd
    for i, (n, p) in enumerate(chunks):
        todo.append((at, n, n + p, r["prefill_tables"][i]))
        at += n
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    scores = None if s["scores"] is None else s["scores"].double()
    for first, lq, lk, table in todo:
        k = _double_rows(s, "k", table, lk)
        v = _double_rows(s, "v", table, lk) if case["kind"] == "attend" else None
        hidden = torch.arange(lk, device="cuda")[None] > torch.arange(lk - lq, lk, device="cuda")[:, None]
        weights = torch.zeros(hkv, lk, dtype=torch.float64, device="cuda")
        for h in range(case["hq"]):
            j = h // (case["hq"] // hkv)
            z = (s["q"][first:first + lq, h].double() @ k[:, j].T) / math.sqrt(HD)
            p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            if v is not None:
                out[first:first + lq, h] = p @ v[:, j]
            weights[j] += p.sum(0)
        if scores is not None:
            place = torch.arange(lk, device="cuda")
            page = table.long()[place // case["block"]]
            old = scores[page, :, place % case["block"]].T
            old = torch.where(place[None] >= lk - lq, 0.0, old)
            scores[page, :, place % case["block"]] = (old + weights).T
    return out if scores is None else scores


def _exact_evict(s):
    c = s["case"]
    block, budget, recent, hkv = c["block"], c["budget"], c["recent"], c["hkv"]
    lens = _lens(c)
    live = s["scores"].double().cpu()
    tables = s["tables"].long().cpu()
    kept = torch.full((c["layers"], len(lens), hkv, budget), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        place = torch.arange(n)
        page, at = tables[r][place // block], place % block
        w = live[:, page, :, at].permute(1, 2, 0).contiguous() if n else None   # [layers, kv_heads, n]
        if n <= budget:
            kept[:, r, :, :n] = place.int()
            continue
        old = n - recent
        heavy = torch.sort(-w[..., :old], dim=-1, stable=True).indices[..., :budget - recent]
        chosen = torch.cat((heavy.sort(-1).values, torch.arange(old, n).expand(c["layers"], hkv, recent)), -1)
        kept[:, r] = chosen.int()
        w2 = torch.zeros_like(w)
        w2[..., :budget] = torch.gather(w, -1, chosen)
        live[:, page, :, at] = w2.permute(2, 0, 1)
    return torch.tensor([min(n, budget) for n in lens]), kept, live, None, None
