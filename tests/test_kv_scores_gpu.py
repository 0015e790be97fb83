"""Accumulated attention weights and eviction on the GPU against the 64-bit
definition (oracle/kv_scores.py), and a serving run that uses both with a
4-bit pool."""
import numpy as np
import pytest
import torch

import slo_attn
from fp4_cases import D, Rows, i32, random_values
from oracle import kv_scores
from test_fp4_gpu import CASES

pytestmark = pytest.mark.gpu


def weigh(case, device, scores, **over):
    kc, vc, ks, vs = case.pool.device(device)
    slo_attn.accumulate_attention(case.q.to(device), kc, scores, case.scale, num_kv_heads=case.hkv, k_scale=ks,
                                  **{**case.arguments(device), **over})
    return scores


def expected(case, start):
    """(scores, bound of their error) in 64 bits.

    A weight's relative error: that of its logit and of its row's sum (see
    Rows.attend), the sum's own n additions, the rounding of the log2-sum, and
    the sum over the row's queries and the group; the sum added to the score
    rounds once more."""
    want, bound = start.double().clone(), torch.zeros_like(start, dtype=torch.float64)
    _, weights, _ = case.attend()
    group = case.hq // case.hkv
    for (first, n, m, table), (w, fp32) in zip(case.rows(), weights):
        m = max(m, 0)
        top = 1.5 * fp32 * 2.0 ** 24 / (D + 4)  # log2 units of the largest logit, at least
        rel = fp32 + 2.0 ** -24 * (m / 16 + n * group + 64 + 4 * top)
        kv_scores.accumulate(want, w, table, max(m - n, 0), case.block)
        grow = torch.zeros_like(bound)
        kv_scores.accumulate(grow, w * rel[..., None], table, 0 if n >= m else m - n, case.block)
        bound += grow
    return want, bound + 2.0 ** -23 * want.abs() + 1e-30


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("name", CASES)
def test_weights_of_every_row_shape(device, fmt, name):
    case = Rows(fmt, **{"seed": len(name), **CASES[name]})
    start = torch.rand(case.blocks, case.hkv, case.block, generator=torch.Generator().manual_seed(2))
    want, bound = expected(case, start)
    got = weigh(case, device, start.to(device)).double().cpu()
    off = (got - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), f"{(off / bound).max():.3f} of the bound"


def test_stale_scores_of_new_tokens_are_replaced(device):
    case = Rows("bf16", [65, 10], [(20, 44), (30, 0)], hq=8, hkv=2, seed=3)
    start = torch.full((case.blocks, 2, case.block), float("nan"))
    for _, n, m, table in case.rows():
        for j in range(m - n):
            start[table[j // case.block], :, j % case.block] = 0.0
    got = weigh(case, device, start.to(device)).cpu()
    for _, n, m, table in case.rows():
        row = torch.stack([got[table[j // case.block], :, j % case.block] for j in range(m)])
        # every query of every head gives a weight of 1 in all
        assert torch.allclose(row.sum(0), torch.full((2,), float(n * 4)), rtol=1e-4)
    live = sum(m for _, _, m, _ in case.rows()) * 2
    assert torch.isnan(got).sum() == got.numel() - live


def test_phases_and_repeats_add_up(device):
    case = Rows("fp4", [300, 33], [(50, 70)], hq=16, hkv=4, seed=5)
    zero = torch.zeros(case.blocks, 4, case.block, device=device)
    both = weigh(case, device, zero.clone())
    apart = weigh(case, device, weigh(case, device, zero.clone(), phases=1), phases=2)
    assert torch.equal(both, apart)
    twice = weigh(case, device, both.clone())
    for _, n, m, table in case.rows():
        for j in range(m):
            a, b = both[table[j // case.block], :, j % case.block], twice[table[j // case.block], :, j % case.block]
            assert torch.equal(b, a + a if j < m - n else a)


def test_rows_that_share_a_prefix_both_count(device):
    case = Rows("bf16", [90, 75, 130], hq=8, hkv=2, block=64, seed=6)
    case.tables[1][0] = case.tables[2][0] = case.tables[0][0]
    start = torch.zeros(case.blocks, 2, 64)
    want, bound = expected(case, start)
    got = weigh(case, device, start.to(device)).double().cpu()
    assert ((got - want).abs() <= bound + 3 * 2.0 ** -24 * want).all()


# ---------------------------------------------------------------- eviction
def evict_case(fmt, lens, budget, recent, hkv, block, layers, seed, device, d=D, special=False):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    blocks = sum(pages) + 2
    order, at, tables = torch.randperm(blocks, generator=g).tolist(), 0, []
    for n in pages:
        tables.append(order[at:at + n] + [-1] * (max(pages + [1]) - n))
        at += n
    width = {"bf16": 2 * d, "fp8": d, "fp4": d // 2}[fmt]
    by_head = fmt == "fp4"
    shape = (layers, blocks, hkv, block) if by_head else (layers, blocks, block, hkv)
    raw = [torch.randint(0, 256, (*shape, width), generator=g, dtype=torch.uint8) for _ in range(2)]
    if fmt == "fp4":
        scale = [torch.randint(63, 190, (*shape, d // 32), generator=g, dtype=torch.uint8) for _ in range(2)]
    else:
        scale = [torch.rand(shape, generator=g) if fmt == "fp8" else None for _ in range(2)]
    scores = (torch.randint(0, 12, (layers, blocks, hkv, block), generator=g).float() - 3) * 0.25  # many ties
    if special:
        pick = torch.rand(scores.shape, generator=g)
        scores[pick < 0.1] = float("nan")
        scores[(pick > 0.1) & (pick < 0.15)] = float("inf")
        scores[(pick > 0.15) & (pick < 0.2)] = -float("inf")
        scores[(pick > 0.2) & (pick < 0.3)] = -0.0
    typed = [t.to(device).view({"bf16": torch.bfloat16, "fp8": torch.uint8, "fp4": torch.float4_e2m1fn_x2}[fmt]) for t in raw]
    dev = dict(k=typed[0], v=typed[1], scores=scores.to(device), ks=None if scale[0] is None else scale[0].to(device),
               vs=None if scale[1] is None else scale[1].to(device), lens=i32(lens, device), tables=i32(tables, device))
    # what is expected, by copies of rows
    want_kept = torch.full((layers, len(lens), hkv, budget), -1, dtype=torch.int32)
    arrays = [t.clone() for t in (*raw, *(s for s in scale if s is not None))]
    new_scores = scores.clone()
    for l in range(layers):
        for r, n in enumerate(lens):
            for h in range(hkv):
                place = [(tables[r][j // block], j % block) for j in range(n)]
                w = np.array([float(scores[l, p, h, o]) for p, o in place])
                kept = kv_scores.choose(w, budget, recent)
                want_kept[l, r, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
                if n <= budget:
                    continue
                for a, src in zip(arrays, (*raw, *(s for s in scale if s is not None))):
                    for i, j in enumerate(kept):
                        (p, o), (p2, o2) = place[j], place[i]
                        a[(l, p2, h, o2) if by_head else (l, p2, o2, h)] = src[(l, p, h, o) if by_head else (l, p, o, h)]
                for i, (p, o) in enumerate(place):
                    new_scores[l, p, h, o] = scores[l, place[kept[i]][0], h, place[kept[i]][1]] if i < budget else 0.0
    return dev, want_kept, arrays, new_scores


def run_evict(dev, budget, recent, layered):
    pick = (lambda t: t) if layered else (lambda t: None if t is None else t[0])  # noqa: E731
    return slo_attn.evict_kv(pick(dev["k"]), pick(dev["v"]), pick(dev["scores"]), dev["lens"], dev["tables"], budget, recent,
                             pick(dev["ks"]), pick(dev["vs"]))


EVICT = [
    ("bf16", [100, 64, 63, 1, 0, 65], 64, 16, 2, 64, 1, 128, False),
    ("fp8", [300, 129, 40], 100, 0, 4, 64, 2, 128, False),
    ("fp4", [300, 129, 500, 5], 33, 33, 2, 128, 3, 128, False),
    ("bf16", [40, 3, 2], 1, 1, 1, 64, 2, 64, False),
    ("fp4", [90, 200], 77, 5, 3, 192, 2, 64, True),
    ("fp8", [200, 130], 90, 7, 2, 64, 1, 256, True),
    ("fp4", [2500, 1200], 1025, 100, 1, 256, 1, 128, True),
    ("bf16", [1300], 1299, 1000, 2, 256, 1, 128, False),
]


@pytest.mark.parametrize("fmt,lens,budget,recent,hkv,block,layers,d,special", EVICT)
def test_eviction_keeps_the_newest_and_the_heaviest(device, fmt, lens, budget, recent, hkv, block, layers, d, special):
    dev, kept, arrays, scores = evict_case(fmt, lens, budget, recent, hkv, block, layers, len(lens) + budget, device, d, special)
    new_lens, got = run_evict(dev, budget, recent, layers > 1)
    assert new_lens.tolist() == [min(n, budget) for n in lens]
    assert torch.equal(got.cpu().view(kept.shape), kept)
    have = [dev["k"], dev["v"]] + [s for s in (dev["ks"], dev["vs"]) if s is not None]
    for h, want in zip(have, arrays):
        assert torch.equal(h.cpu().view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(dev["scores"].cpu().view(torch.int32), scores.view(torch.int32))


def test_eviction_of_a_long_row(device):
    # above the 32,768 tokens that a selection could hold at 32 a thread
    dev, kept, arrays, scores = evict_case("fp4", [40001], 700, 50, 1, 256, 1, 12, device)
    _, got = run_evict(dev, 700, 50, False)
    assert torch.equal(got.cpu().view(kept.shape), kept)
    assert torch.equal(dev["k"].cpu().view(torch.uint8), arrays[0])
    assert torch.equal(dev["scores"].cpu(), scores)


def test_tokens_in_no_page_go_first_and_do_not_move(device):
    dev, _, _, _ = evict_case("bf16", [200, 130], 60, 10, 2, 64, 1, 5, device)
    dev["scores"].abs_().add_(0.5)
    dev["tables"][0, 1] = -1
    dev["tables"][1, 2] = 10 ** 7  # the row's newest tokens: kept, but in no page
    before = dev["k"].clone()
    lens, kept = run_evict(dev, 60, 10, False)
    kept = kept.cpu()
    assert lens.tolist() == [60, 60]
    assert not ((kept[0] >= 64) & (kept[0] < 128)).any()
    assert (kept[1][:, -2:] == torch.tensor([128, 129])).all()
    page = int(dev["tables"][1, 0])
    for h in range(2):
        for i in range(60):
            j = int(kept[1, h, i])
            old = before[0, page, i, h] if j >= 128 else before[0, int(dev["tables"][1, j // 64]), j % 64, h]
            assert torch.equal(dev["k"][0, page, i, h].view(torch.int16), old.view(torch.int16))


def test_refusals(device):
    dev, _, _, _ = evict_case("fp8", [100], 60, 10, 2, 64, 2, 5, device)
    for error, over in ((ValueError, dict(budget=0)), (ValueError, dict(recent=61)), (ValueError, dict(recent=-1)),
                        (ValueError, dict(ks=None)), (ValueError, dict(scores=dev["scores"][0])),
                        (TypeError, dict(lens=dev["lens"].long())), (ValueError, dict(lens=dev["lens"].repeat(2))),
                        (ValueError, dict(scores=dev["scores"].transpose(2, 3))), (ValueError, dict(v=dev["v"][:, :1]))):
        a = {**dev, "budget": 60, "recent": 10, **over}
        with pytest.raises(error):
            slo_attn.evict_kv(a["k"], a["v"], a["scores"], a["lens"], a["tables"], a["budget"], a["recent"], a["ks"], a["vs"])
    case = Rows("bf16", [40], [(3, 10)], hq=8, hkv=2)
    s = torch.zeros(case.blocks, 2, 64, device=device)
    for error, over in ((ValueError, dict(prefill_tables=None)), (ValueError, dict(num_decode=9))):
        with pytest.raises(error):
            weigh(case, device, s, **over)
    with pytest.raises(ValueError):
        weigh(case, device, s[:, :, :32])
    with pytest.raises(TypeError):
        weigh(case, device, s.double())
    with pytest.raises(RuntimeError, match="track_scores"):
        slo_attn.KVPool(1, 2, 64, 1, D, "fp4_e2m1", device).evict(i32([3], device), i32([[0]], device), 2, 1)


# ------------------------------------------------------------- all together
@pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3fn", "fp4_e2m1"])
def test_serving_run_with_eviction(device, fmt):
    """A prompt in two chunks, decode steps, eviction whenever a row passes its budget, and further steps: outputs
    against attention in 64 bits over the tokens that a plain bookkeeping says are left."""
    hq, hkv, block, layers, budget, recent = 8, 2, 64, 2, 96, 24
    pool = slo_attn.KVPool(layers, 9, block, hkv, D, fmt, device, track_scores=True)
    model = [slo_attn.Attention(hq, D, D ** -0.5, hkv) for _ in range(layers)]
    pool.attach(model)
    g = torch.Generator().manual_seed(13)
    tables = [[5, 0, 3], [8, 1, 4]]
    lens = [0, 0]
    left = [[[([], []) for _ in range(hkv)] for _ in range(2)] for _ in range(layers)]  # per layer, row, head: K and V rows
    weight = [[[[] for _ in range(hkv)] for _ in range(2)] for _ in range(layers)]
    evictions = 0
    for step, news in enumerate([(60, 17), (55, 0)] + [(1, 1)] * 60):
        n = sum(news)
        q, k, v = (random_values(g, n, h, D) for h in (hq, hkv, hkv))
        slots = [tables[r][(lens[r] + i) // block] * block + (lens[r] + i) % block for r in (0, 1) for i in range(news[r])]
        lens = [a + b for a, b in zip(lens, news)]
        if step < 2:
            ends = [news[0], n]
            meta = slo_attn.MixedAttentionContext(0, n, None, None, i32([0, *ends], device), i32([0, lens[0], sum(lens)], device),
                                                  i32(tables, device), max(news), max(lens), True)
        else:
            meta = slo_attn.MixedAttentionContext(2, 0, i32(lens, device), i32(tables, device), None, None, None, 0, 0, False)
        slo_attn.set_context(False, slot_mapping=i32(slots, device), mixed=meta)
        for l, layer in enumerate(model):
            out = layer(q.to(device), k.to(device), v.to(device)).double().cpu()
            kq, vq = (t.double().cpu() for t in pool.read(l, i32(slots, device)))
            at = 0
            for r in (0, 1):
                for h in range(hkv):
                    kk, vv = left[l][r][h]
                    kk.extend(kq[at:at + news[r], h])
                    vv.extend(vq[at:at + news[r], h])
                    weight[l][r][h].extend([0.0] * news[r])
                    if not news[r]:
                        continue
                    m = lens[r]
                    o, w, size, logit = kv_scores.attend(q[at:at + news[r], 4 * h:4 * h + 4].double(), torch.stack(kk)[:, None],
                                                         torch.stack(vv)[:, None], m - news[r], D ** -0.5)
                    weight[l][r][h] = (torch.tensor(weight[l][r][h], dtype=torch.float64) + w.sum((0, 1))).tolist()
                    # decode: outputs and codes as in Rows.attend; E4M3FN values read back in bf16 are off by 2^-8 too
                    tol = 2.0 ** -8 * (3 if fmt == "fp8_e4m3fn" else 1) * (size + 2 * o.abs())
                    tol = tol + 2 * 2.0 ** -8 * logit[..., None] * D ** -0.5 * (size + o.abs()) * (fmt == "fp8_e4m3fn")
                    assert ((out[at:at + news[r], 4 * h:4 * h + 4] - o).abs() <= 1.05 * tol + 1e-4).all()
                at += news[r]
        slo_attn.reset_context()
        if max(lens) > budget + 8:
            new_lens, kept = pool.evict(i32(lens, device), i32(tables, device), budget, recent)
            evictions += 1
            kept = kept.cpu()
            for l in range(layers):
                for r in (0, 1):
                    for h in range(hkv):
                        places = [j for j in kept[l, r, h].tolist() if j >= 0]
                        w = weight[l][r][h]
                        if lens[r] > budget:
                            assert places[-recent:] == list(range(lens[r] - recent, lens[r])) and len(places) == budget
                            # no token that went weighed clearly more than one that stayed
                            gone = set(range(lens[r] - recent)) - set(places)
                            low = min(w[j] for j in places[:-recent])
                            assert max(w[j] for j in gone) <= low * (1 + (0.05 if fmt == "fp8_e4m3fn" else 1e-3)) + 1e-4
                        left[l][r][h] = tuple([x[j] for j in places] for x in left[l][r][h])
                        weight[l][r][h] = [w[j] for j in places]
            lens = new_lens.tolist()
    assert evictions >= 3
