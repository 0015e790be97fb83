"""Attention with a sliding window and sinks on the GPU against the 64-bit
definition (oracle/window.py), over pools of every format and cold rows."""
import pytest
import torch

import slo_attn
from fp4_cases import D, i32, random_values
from oracle import window as owin
from window_cases import WindowRows

pytestmark = pytest.mark.gpu


def call(case, device, q=None, **over):
    kc, vc, ks, vs = case.pool.device(device)
    args = dict(num_kv_heads=case.hkv, k_scale=ks, v_scale=vs, window=case.window, sinks=case.sinks, **case.arguments(device))
    return slo_attn.paged_attention(case.q.to(device) if q is None else q, kc, vc, case.scale, **{**args, **over})


def check(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), f"{(off / bound).max():.3f} of the bound"


CASES = {
    "one_key": dict(lens=[1], window=1, sinks=0),
    "own_key_only": dict(lens=[5, 64, 65, 300], chunks=[(70, 0), (3, 99)], window=1, sinks=0),
    "own_key_and_the_first": dict(lens=[5, 64, 65, 300], chunks=[(70, 0), (3, 99)], window=1, sinks=1),
    "empty_rows": dict(lens=[0, 1, 0, 31, 32, 33, 63, 64, 65, 0], window=32, sinks=3),
    "window_of_a_tile": dict(lens=[63, 64, 65, 127, 128, 129, 200], chunks=[(64, 64), (65, 63)], window=64, sinks=0),
    "window_past_every_row": dict(lens=[30, 200], chunks=[(40, 60)], window=1 << 30, sinks=1 << 30),
    "sinks_past_the_row": dict(lens=[30, 200], chunks=[(40, 60)], window=5, sinks=500),
    "sinks_end_inside_a_tile": dict(lens=[700, 900], chunks=[(50, 600), (9, 1000)], window=77, sinks=130, block=128),
    "sinks_meet_the_window": dict(lens=[140, 141, 142, 150], chunks=[(30, 130)], window=70, sinks=70),
    "no_sinks": dict(lens=[333, 80], chunks=[(70, 400)], window=50, sinks=0, block=192),
    "split_rows": dict(lens=[3000, 17, 1023, 2049], hq=8, hkv=2, gain=2.0, window=1500, sinks=70),
    "group_1": dict(lens=[70, 200], chunks=[(150, 20)], hq=2, hkv=2, block=192, window=61, sinks=2),
    "group_5": dict(lens=[70, 300], chunks=[(33, 200)], hq=10, hkv=2, gain=3.0, window=90),
    "group_7_prefill": dict(lens=[90], chunks=[(37, 0), (5, 100), (1, 0)], hq=28, hkv=4, window=20),
    "group_16": dict(lens=[333], chunks=[(20, 145)], hq=16, hkv=1, block=256, window=65, sinks=1),
    "peaked": dict(lens=[400, 900], chunks=[(70, 130)], hq=8, hkv=2, gain=30.0, window=150),
    "chunks": dict(lens=[], chunks=[(64, 0), (33, 64), (130, 701), (1, 511), (3, 0)], hq=16, hkv=4, window=128, sinks=5),
    "fewer_keys_than_queries": dict(lens=[], chunks=[(40, -7), (20, -20), (9, 3)], hq=8, hkv=2, window=6, sinks=2),
    "split_tiles": dict(lens=[], chunks=[(3, 2600), (40, 1700)], hq=8, hkv=2, window=2000, sinks=9),
    "mixed": dict(lens=[5, 700, 64], chunks=[(100, 0), (50, 333)], block=256, window=99),
    "negative_scale": dict(lens=[80], chunks=[(30, 20)], hq=8, hkv=2, scale=-0.11, window=33),
    "many_rows": dict(lens=[(37 * i) % 130 for i in range(150)], chunks=[(i % 5, 3 * i) for i in range(70)], hq=4, hkv=2,
                      window=41, sinks=7),
    "many_tiles": dict(lens=[], chunks=[(700, 30), (40, 0)], hq=16, hkv=1, window=100),
    "tables_far_wider_than_the_rows": dict(lens=[100, 5, 0], chunks=[(9, 70), (2, 0)], hq=8, hkv=2, spare=90, window=50),
    "pages_not_in_the_pool": dict(lens=[200, 60], chunks=[(20, 140)], hq=8, hkv=2, window=100, sinks=10, give_back=False,
                                  holes=[(0, 2, -1), (1, 0, 10 ** 6), (2, 0, -5), (2, 1, 1 << 30)]),
}


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("name", CASES)
def test_attention_under_a_window(device, name, fmt):
    case = WindowRows(fmt, **{"seed": len(name), **CASES[name]})
    check(call(case, device), *case.attend())


@pytest.mark.parametrize("name", ["chunks", "own_key_only", "group_7_prefill", "many_tiles", "fewer_keys_than_queries", "group_1"])
def test_cold_rows_under_a_window(device, name):
    # rows without tables, read from views of a wider projection; a row's keys end at the next one's
    over = {**CASES[name], "lens": []}
    over["chunks"] = [(n, min(p, 0)) for n, p in over["chunks"]] + [(77, -1)]
    case = WindowRows("bf16", give_back=False, seed=3, **over)
    k, v = (torch.cat([case.pool.values(t, max(m, 0), side)[0] for _, _, m, t in case.rows()]).to(torch.bfloat16) for side in (0, 1))
    wide = torch.full((len(k), 2 * case.hkv + 3, D), float("nan"), dtype=torch.bfloat16, device=device)
    wide[:, 1:1 + case.hkv], wide[:, 2 + case.hkv:2 + 2 * case.hkv] = k.to(device), v.to(device)
    args = {**case.arguments(device), "prefill_tables": None}
    got = slo_attn.paged_attention(case.q.to(device), None, None, case.scale, num_kv_heads=case.hkv, window=case.window,
                                   sinks=case.sinks, k=wide[:, 1:1 + case.hkv], v=wide[:, 2 + case.hkv:2 + 2 * case.hkv], **args)
    check(got, *case.attend())


@pytest.mark.parametrize("rows", [1, 11])  # tiles of two halves, and of one
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4", "cold"])
def test_rounding_of_a_dominating_weight_cancels(device, fmt, rows):
    """One late key has nearly all of every query's weight, which is some number between 90 and 190 times the first key's.

    Weights w are rounded to bf16, w' = w (1 + d) with |d| <= 2^-8, and an fp32 logit moves a weight by
    2 (D + 4) 2^-24 sum|q k| scale = f more.  The outputs sum(w' v) / sum(w') are off by
    sum(w' (v - o)) / sum(w'), at most (2^-8 + f) sum p|v - o| / (1 - 2^-8 - f) for normalised weights p; sums of 300 products
    in fp32 by 300 2^-24 of their size, the sum's own (E4M3FN: a reciprocal of three terms) by as much again; the result
    is rounded once, 2^-8."""
    n, prefix, late, hq, hkv, scale = 100, 200, 150, 32, 2, 5 / 512
    case = WindowRows("bf16" if fmt == "cold" else fmt, [], [(n, prefix)] * rows, hq=hq, hkv=hkv, seed=8, window=1000, sinks=0,
                      scale=scale, give_back=False)
    g = torch.Generator().manual_seed(12)
    signs = 2.0 * torch.randint(0, 2, (hkv, D), generator=g) - 1
    size = torch.full((n + prefix, 1, 1), -8.0)
    size[0], size[late] = 0.0, 4.0
    k = (size * signs).to(torch.bfloat16)
    vs = [random_values(g, n + prefix, hkv, D) for _ in range(rows)]
    case.q = ((0.9 + 0.15 * torch.rand(rows * n, hq, 1, generator=g)) * signs.repeat_interleave(hq // hkv, 0)).to(torch.bfloat16)
    for (_, _, _, table), v in zip(case.rows(), vs):
        case.pool.write(table, k, v)
    if fmt == "cold":
        kk, vv = k.repeat(rows, 1, 1).to(device), torch.cat(vs).to(device)
        got = call(case, device, k=kk, v=vv, prefill_tables=None)
    else:
        got = call(case, device)
    unseen = torch.ones(n, n + prefix, dtype=torch.bool).triu(prefix + 1)
    for first, _, m, table in case.rows():
        (k64, _), (v64, _) = (case.pool.values(table, m, side) for side in (0, 1))
        q64 = case.q[first:first + n].double()
        for h in range(hq):
            kh, vh = k64[:, h // (hq // hkv)], v64[:, h // (hq // hkv)]
            p = torch.softmax((q64[:, h] @ kh.T * scale).masked_fill(unseen, float("-inf")), -1)
            assert (p[:, late] > 0.98).all() and (p[:, late] < 191 * p[:, 0]).all() and (p[:, late] > 85 * p[:, 0]).all()
            o = p @ vh
            apart = torch.stack([(w[:, None] * (vh - x).abs()).sum(0) for w, x in zip(p, o)])
            moved = 2.0 ** -8 + 2 * (D + 4) * 2.0 ** -24 * (q64[:, h].abs() @ kh.abs().T).max() * scale
            bound = 2.0 ** -8 * o.abs() + moved * apart / (1 - moved) * (1 + 2.0 ** -8) + 700 * 2.0 ** -24 * (p @ vh.abs() + o.abs())
            check(got[first:first + n, h], o, bound)


def test_scales_that_make_nothing_of_values(device):
    # E4M3FN V scales of 0, or so small that no bf16 output shows them, leave a key its weight; a negative one turns its values
    case = WindowRows("fp8", [], [(90, 40)], hq=8, hkv=2, seed=6, window=50, sinks=2, give_back=False)
    table = case.tables[0]
    for j, x in ((0, 0.0), (30, 2.0 ** -120), (70, 0.0), (71, 2.0 ** -99), (100, -0.5), (129, 0.0)):
        case.pool.scale[1][table[j // case.block], j % case.block] = x
    check(call(case, device), *case.attend())


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_cold_rows_beside_decode_rows_of_a_pool(device, fmt):
    case = WindowRows(fmt, [70, 5], [(33, 0), (150, 0)], hq=16, hkv=4, seed=5, window=40)
    g = torch.Generator().manual_seed(1)
    k, v = (random_values(g, 183, 4, D) for _ in range(2))
    got = call(case, device, k=k.to(device), v=v.to(device), prefill_tables=None)
    want, bound = case.attend()
    check(got[:2], want[:2], bound[:2])
    at = 0
    for n in (33, 150):
        o, size, logit = owin.attend(case.q[2 + at:2 + at + n].double(), k[at:at + n].double(), v[at:at + n].double(), 0,
                                     case.scale, 40, 4)
        spread = size + o.abs()
        lim = (2.0 ** -8 * (spread + o.abs()) + (2 * (D + 4) * 2.0 ** -24 * logit * case.scale)[..., None] * spread) * 1.02
        check(got[2 + at:2 + at + n], o, lim)
        at += n
    # rows and cu_seqlens that claim more keys than there are rows of k and v read no further
    args = case.arguments(device)
    args["prefill_cu_k"] = i32([0, 33, 5000], device)
    call(case, device, k=k.to(device), v=v.to(device), **{**args, "prefill_tables": None})


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_a_window_past_every_key_is_plain_attention(device, fmt):
    # within the two calls' bounds of the same 64-bit result
    case = WindowRows(fmt, [300, 5, 64], [(70, 200), (20, 0)], hq=16, hkv=4, seed=2, window=4096, sinks=0)
    check(call(case, device, window=0), *case.attend())
    check(call(case, device), *case.attend())


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_views_phases_and_rows_past_every_row(device, fmt):
    case = WindowRows(fmt, [100, 30], [(17, 40), (5, 0)], hq=8, hkv=2, seed=4, window=23)
    want, bound = case.attend()
    nan = torch.full((40, 8, D), float("nan"), dtype=torch.bfloat16)
    wide = torch.zeros(case.tokens + 40, 12, D, dtype=torch.bfloat16, device=device)
    wide[:, :8] = torch.cat((case.q, nan)).to(device)
    for phases in (1, 2, 3):
        out = torch.full((case.tokens + 42, 10, D), 7.0, dtype=torch.bfloat16, device=device)
        got = call(case, device, q=wide[:, :8], out=out[:case.tokens + 40, :8], phases=phases, max_q=60, max_k=5000)
        assert got.data_ptr() == out.data_ptr()
        assert (out[case.tokens + 40:] == 7).all() and (out[:, 8:] == 7).all() and not got[case.tokens:].any()
        for bit, rows in ((1, slice(0, 2)), (2, slice(2, case.tokens))):
            if phases & bit:
                check(got[rows], want[rows], bound[rows])
            else:
                assert (got[rows] == 7).all()


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_captured_step_replays(device, fmt):
    # lengths, chunks and tables change between replays, eager calls in between
    case = WindowRows(fmt, [1500, 40, 700], [(20, 300)], hq=16, hkv=4, seed=11, window=600, give_back=False)
    kc, vc, ks, vs = case.pool.device(device)
    args = case.arguments(device)
    q = case.q.to(device)

    def step():
        return slo_attn.paged_attention(q, kc, vc, case.scale, num_kv_heads=4, k_scale=ks, v_scale=vs, window=600, sinks=4, **args)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lens, cu_q, cu_k in (([1500, 40, 700], [0, 20], [0, 320]), ([1, 0, 699], [0, 1], [0, 1]), ([777, 33, 64], [0, 0], [0, 0]),
                             ([1500, 40, 700], [0, 20], [0, 320])):
        args["decode_lens"].copy_(i32(lens, device))
        args["prefill_cu_q"].copy_(i32(cu_q, device))
        args["prefill_cu_k"].copy_(i32(cu_k, device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step())


def test_two_captured_graphs_replay_at_once(device):
    # each graph has its own workspace: cut decode rows, halves of tiles and cut tiles
    cases = [WindowRows("bf16", [2500, 900], [(60, 1900)], hq=8, hkv=2, seed=s, window=1800) for s in (31, 32)]
    states = [(c.q.to(device), c.pool.device(device), c.arguments(device)) for c in cases]

    def run(i):
        q, (kc, vc, _, _), args = states[i]
        return slo_attn.paged_attention(q, kc, vc, cases[i].scale, num_kv_heads=2, window=1800, sinks=4, **args)

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [None, None]
    for i in (0, 1):
        with torch.cuda.graph(graphs[i]):
            got[i] = run(i)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        run(0)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3fn"])
def test_captured_mixed_steps_of_windowed_layers(device, fmt):
    # a bucket's graph (metadata, store, attention; padded rows and tokens) against the same bucket run eagerly
    hq, hkv, block, width = 8, 2, 64, 6
    pool = slo_attn.KVPool(2, 24, block, hkv, D, fmt, device)
    layers = [slo_attn.Attention(hq, D, D ** -0.5, hkv, window=w, sinks=3) for w in (33, 100)]
    pool.attach(layers)
    g = torch.Generator().manual_seed(3)
    table = random_values(g, 50, hq + 2 * hkv, D).to(device)

    def forward(ids, positions):
        x = table[ids]
        out = 0
        for layer in layers:
            out = out + layer(x[:, :hq].contiguous(), x[:, hq:hq + hkv], x[:, hq + hkv:])
        return out

    buf = slo_attn.MixedStepBuffers(4, 3, 150, width, block, width * block, device)
    graph = slo_attn.MixedStepGraph(buf, forward, exact_history=fmt != "bf16")
    pool.kv.zero_()
    rows = [[0, 1, 7], [2], [5], [6]]
    steps = [([], [(0, 60), (0, 33)], [[0, 1], [2]], [i % 50 for i in range(93)]),
             ([60, 33], [(0, 20)], [[0, 1], [2], [5]], list(range(22))),
             ([61, 34, 20], [(0, 1)], [[0, 1], [2], [5], [6]], [1, 2, 3, 4]),
             ([35, 21], [(62, 100)], [[2], [5], rows[0]], [i % 50 for i in range(102)])]
    for step in steps:
        before = pool.kv.clone(), None if pool.scale is None else pool.scale.clone()
        got = graph.run(*step).clone()
        torch.cuda.synchronize()
        after = pool.kv.clone()
        pool.kv.copy_(before[0])
        if before[1] is not None:
            pool.scale.copy_(before[1])
        buf.build()
        buf.set_context(fmt == "bf16" or any(s for s, n in step[1] if n))
        want = forward(buf.input_ids, buf.positions)
        slo_attn.reset_context()
        assert torch.isfinite(want).all() and torch.equal(got, want) and torch.equal(after, pool.kv)


def test_rows_do_not_depend_on_their_neighbours(device):
    # a row alone takes other launch shapes (halves, cuts) than among many: both within the bound of the same result
    case = WindowRows("bf16", [1200, 700] * 20, [(50, 600), (33, 0)] * 6, hq=16, hkv=4, seed=6, window=500)
    want, bound = case.attend()
    check(call(case, device), want, bound)
    one = WindowRows("bf16", [], [(50, 600)], hq=16, hkv=4, seed=7, window=500)
    check(call(one, device), *one.attend())


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_a_row_alone_is_what_it_is_among_others(device, fmt):
    # the same queries, pages and keys in a call of their own, which cuts decode rows and tiles further: within the bound
    # of the one definition both times, and so within twice that of each other
    base = WindowRows(fmt, [2200, 700], [(50, 2600), (33, 0)], hq=16, hkv=4, seed=6, window=1500)
    base.q = torch.randn(311, 16, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    case = base.part([2200, 700] * 31, base.chunks * 3, base.tables[:2] * 31 + base.tables[2:] * 3, slice(0, 311))
    among = call(case, device)
    first = len(case.lens)
    for lens, chunks, row, queries in (([2200], [], 6, slice(6, 7)), ([700], [], 61, slice(61, 62)),
                                       ([], [(50, 2600)], first + 2, slice(first + 83, first + 133)),
                                       ([], [(33, 0)], first + 5, slice(first + 216, first + 249)),
                                       ([2200, 700], [], slice(2, 4), slice(2, 4))):
        one = case.part(lens, chunks, case.tables[row] if isinstance(row, slice) else [case.tables[row]], queries)
        want, bound = one.attend()
        alone = call(one, device)
        check(alone, want, bound)
        check(among[queries], want, bound)
        check(alone, among[queries].double().cpu(), 2 * bound)


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_each_replay_is_the_definition_of_its_step(device, fmt):
    # a captured call with rows shorter than the plan's, empty ones, and fewer queries than its capacity, each replay against
    # the 64-bit result for the lengths of that replay; query rows past the last row are zeros
    case = WindowRows(fmt, [1500, 40, 700], [(20, 300)], hq=16, hkv=4, seed=11, window=600, give_back=False)
    kc, vc, ks, vs = case.pool.device(device)
    args = case.arguments(device)
    q = case.q.to(device)
    out = torch.empty_like(q)

    def step():
        slo_attn.paged_attention(q, kc, vc, case.scale, num_kv_heads=4, k_scale=ks, v_scale=vs, window=600, sinks=4, out=out, **args)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens, (n, prefix) in (([1500, 40, 700], (20, 300)), ([1, 0, 699], (1, 0)), ([777, 33, 64], (0, 0)), ([0, 0, 0], (19, 301)),
                              ([1400, 39, 1], (7, 200)), ([1500, 40, 700], (20, 300))):
        args["decode_lens"].copy_(i32(lens, device))
        args["prefill_cu_q"].copy_(i32([0, n], device))
        args["prefill_cu_k"].copy_(i32([0, n + prefix], device))
        out.fill_(float("nan"))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        one = case.part(lens, [(n, prefix)], case.tables, slice(0, 3 + n))
        check(got[:3 + n], *one.attend())
        assert not got[3 + n:].any()
        for row, keys in enumerate(lens):
            assert keys or not got[row].any()
        step()
        assert torch.equal(got, out)


def test_two_streams_at_once(device):
    cases = [WindowRows("bf16", [2500, 300], [(60, 900)], hq=16, hkv=4, seed=s, window=1400) for s in (21, 22)]
    states = [(c.q.to(device), c.pool.device(device), c.arguments(device)) for c in cases]

    def run(i):
        q, (kc, vc, _, _), args = states[i]
        return slo_attn.paged_attention(q, kc, vc, cases[i].scale, num_kv_heads=4, window=1400, sinks=4, **args)

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = run(i)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_pool_past_4_gib(device, fmt):
    blocks, block, hkv = {"bf16": 9000, "fp8": 17000, "fp4": 33000}[fmt], 256, 8
    case = WindowRows(fmt, [600, 40], [(10, 400)], hq=16, hkv=hkv, block=block, seed=9, window=200, give_back=False)
    small = call(case, device)
    big = []
    for t in case.pool.device(device):
        if t is None:
            big.append(None)
            continue
        raw = t.view(torch.uint8) if fmt == "fp4" else t
        wide = torch.zeros(blocks, *raw.shape[1:], dtype=raw.dtype, device=device)
        wide[-case.blocks:] = raw
        big.append(wide.view(t.dtype) if fmt == "fp4" else wide)
    case.tables = [[p + blocks - case.blocks if p >= 0 else p for p in t] for t in case.tables]
    got = slo_attn.paged_attention(case.q.to(device), big[0], big[1], case.scale, num_kv_heads=hkv, k_scale=big[2], v_scale=big[3],
                                   window=200, sinks=4, **case.arguments(device))
    assert torch.equal(got, small)


@pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3fn", "fp4_e2m1"])
def test_a_conversation_through_the_layer(device, fmt):
    """A long-context layer as a model runs it: rotation by a scaled table and the KV write in one call, attention with a
    window over the pool, the prompt in two chunks (one of them cold), then tokens one at a time and a mixed step, with
    pages given back behind the window; against the definition on the keys as the pool holds them."""
    hq, hkv, block, window, sinks, n = 16, 4, 64, 100, 5, 400
    pool = slo_attn.KVPool(1, 9, block, hkv, D, fmt, device)
    layer = slo_attn.Attention(hq, D, D ** -0.5, hkv, window=window, sinks=sinks)
    pool.attach([layer])
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(n, (hq + 2 * hkv) * D, generator=g).to(torch.bfloat16).to(device)
    table = slo_attn.rope_cos_sin(D, 4096, 1e4, device, rotary_dim=96,
                                  scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=1024))
    free, row, keys, values, outs, qs = list(range(9)), [], [], [], [], []

    def step(first, count, mode):
        for b in range(-(-(first + count) // block) - len(row)):
            row.append(free.pop())
        slots = i32([row[j // block] * block + j % block for j in range(first, first + count)], device)
        pos = torch.arange(first, first + count, device=device)
        q, k, v = slo_attn.qk_norm_rope_store(qkv[first:first + count], pos, None, None, 0.0, table, hq, hkv, layer.k_cache,
                                              layer.v_cache, slots, *layer._scales(), rotary_dim=96, interleaved=True)
        tables = i32([row], device)
        cu_q, cu_k = i32([0, count], device), i32([0, first + count], device)
        if mode == "prefill":
            slo_attn.set_context(True, cu_q, cu_k, count, first + count, slots, None, tables if first else None)
        elif mode == "decode":
            slo_attn.set_context(False, slot_mapping=slots, context_lens=i32([first + 1], device), block_tables=tables)
        else:
            slo_attn.set_context(False, slot_mapping=slots, mixed=slo_attn.MixedAttentionContext(
                0, count, None, None, cu_q, cu_k, tables, count, first + count, True))
        outs.append(layer(q, k, v, kv_stored=True).reshape(count, hq, D))
        qs.append(q)
        # the second call stores the same bytes again and gives the same bits
        assert torch.equal(layer(q, k, v).reshape(count, hq, D), outs[-1])
        slo_attn.reset_context()
        kk, vv = pool.read(0, slots)
        cold = mode == "prefill" and not first
        keys.append((kk, k if cold else kk))
        values.append((vv, v if cold else vv))
        for b in slo_attn.window_blocks(first + count, window, sinks, block):
            if row[b] >= 0:
                free.append(row[b])
                row[b] = -1

    step(0, 150, "prefill")
    step(150, 130, "prefill")
    for i in range(280, 300):
        step(i, 1, "decode")
    step(300, 100, "mixed")
    assert row.count(-1) >= 3
    at = 0
    for i, (q, o) in enumerate(zip(qs, outs)):
        m = at + len(q)
        k = torch.cat([x[0] for x in keys[:i]] + [keys[i][1]]).double().cpu()
        v = torch.cat([x[0] for x in values[:i]] + [values[i][1]]).double().cpu()
        want, size, logit = owin.attend(q.double().cpu(), k, v, at, D ** -0.5, window, sinks)
        spread = size + want.abs()
        # pool.read rounds E4M3FN values to bf16, which moves a key's logit and a value by 2^-8 of them each
        read = 2.0 ** -8 if fmt == "fp8_e4m3fn" else 0.0
        fp32 = 2 * (D + 4) * 2.0 ** -24 + 2 * read
        bound = (2.0 ** -8 * (spread + want.abs()) + read * size + (torch.expm1(fp32 * logit * D ** -0.5))[..., None] * spread) * 1.02
        check(o, want, bound)
        at = m


def test_cold_rows_as_far_apart_as_they_may_be(device):
    # a row every 64 MiB: a step's offsets pass 2^31; keys that no query sees are anything
    n, keys, hkv, far, window = 40, 134, 2, (1 << 25) - 8, 30
    g = torch.Generator().manual_seed(4)
    q, k, v = random_values(g, n, 8, D), random_values(g, keys, hkv, D), random_values(g, keys, hkv, D)
    k[1:keys - n - window + 1] = v[1:keys - n - window + 1] = float("nan")
    base = torch.empty((keys - 1) * far + 2 * hkv * D, dtype=torch.bfloat16, device=device)
    fk, fv = (base.as_strided((keys, hkv, D), (far, D, 1), i * hkv * D) for i in (0, 1))
    fk.copy_(k)
    fv.copy_(v)
    args = dict(num_kv_heads=hkv, num_prefill=1, prefill_cu_q=i32([0, n], device), prefill_cu_k=i32([0, keys], device), max_q=n,
                max_k=keys, window=window, sinks=1)
    near = slo_attn.paged_attention(q.to(device), None, None, 0.1, k=k.to(device), v=v.to(device), **args)
    got = slo_attn.paged_attention(q.to(device), None, None, 0.1, k=fk, v=fv, **args)
    assert torch.equal(got, near)
    o, size, logit = owin.attend(q.double(), k.double().nan_to_num(), v.double().nan_to_num(), keys - n, 0.1, window, 1)
    spread = size + o.abs()
    check(near, o, (2.0 ** -8 * (spread + o.abs()) + (2 * (D + 4) * 2.0 ** -24 * logit * 0.1)[..., None] * spread) * 1.02)
    with pytest.raises(RuntimeError, match="elements apart"):
        slo_attn.paged_attention(q.to(device), None, None, 0.1, k=base.as_strided((keys - 1, hkv, D), (1 << 25, D, 1)), v=fv, **args)


def test_refusals(device):
    case = WindowRows("bf16", [40], [(3, 10)], hq=8, hkv=2)
    k = torch.zeros(3, 2, D, dtype=torch.bfloat16, device=device)
    q = case.q.to(device)
    for error, over in ((ValueError, dict(window=-1)), (ValueError, dict(window=0, sinks=3)), (ValueError, dict(sinks=-1)),
                        (ValueError, dict(noalloc=True)), (TypeError, dict(q=q.float())), (ValueError, dict(num_kv_heads=4)),
                        (ValueError, dict(prefill_tables=None)), (ValueError, dict(prefill_tables=None, k=k[:, :1], v=k[:, :1])),
                        (ValueError, dict(prefill_tables=None, k=k.float(), v=k)), (ValueError, dict(num_decode=5)),
                        (TypeError, dict(out=torch.empty(4, 8, D, device=device))), (ValueError, dict(out=torch.empty_like(q[:2])))):
        with pytest.raises(error):
            call(case, device, **over)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        case.scale = 0.0
        call(case, device)
    layer = slo_attn.Attention(8, D, 0.1, 2, window=5)
    slo_attn.KVPool(1, 2, 64, 2, D, "bf16", device, track_scores=True).attach([layer])
    with pytest.raises(ValueError, match="kv_scores"):
        layer(q, k, k)
