"""Limits of the compressed KV cache's operators on the GPU: bounds left out or
too small, and what lies past 32 bits."""
import pytest
import torch

import slo_attn
from fp4_cases import D, Rows, i32, random_values
from test_fp4_gpu import CASES
from test_kv_scores_gpu import expected

pytestmark = pytest.mark.gpu

PREFILL = [name for name, case in CASES.items() if case.get("chunks")]
BOUNDS = [dict(), dict(max_q=1, max_k=1), dict(max_q=1 << 16, max_k=1 << 20)]


def without_bounds(case, device):
    return {k: v for k, v in case.arguments(device).items() if k not in ("max_q", "max_k")}


@pytest.mark.parametrize("bounds", BOUNDS, ids=["left_out", "too_small", "too_large"])
@pytest.mark.parametrize("name", PREFILL)
def test_4_bit_attention_does_not_depend_on_the_bounds(device, name, bounds):
    case = Rows("fp4", **{"seed": len(name), **CASES[name]})
    kc, vc, ks, vs = case.pool.device(device)
    got = slo_attn.paged_attention(case.q.to(device), kc, vc, case.scale, num_kv_heads=case.hkv, k_scale=ks, v_scale=vs,
                                   out=torch.full(case.q.shape, float("nan"), dtype=torch.bfloat16, device=device),
                                   **without_bounds(case, device), **bounds)
    want, _, bound = case.attend()
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("bounds", BOUNDS, ids=["left_out", "too_small", "too_large"])
@pytest.mark.parametrize("fmt,name", [(("bf16", "fp8", "fp4")[i % 3], name) for i, name in enumerate(PREFILL)]
                         + [("bf16", "many_tiles"), ("fp8", "chunks"), ("fp4", "pages_not_in_the_pool")])
def test_weights_do_not_depend_on_the_bounds(device, fmt, name, bounds):
    case = Rows(fmt, **{"seed": len(name), **CASES[name]})
    kc, _, ks, _ = case.pool.device(device)
    start = torch.rand(case.blocks, case.hkv, case.block, generator=torch.Generator().manual_seed(2))
    want, bound = expected(case, start)
    got = start.to(device)
    slo_attn.accumulate_attention(case.q.to(device), kc, got, case.scale, num_kv_heads=case.hkv, k_scale=ks,
                                  **without_bounds(case, device), **bounds)
    assert torch.isfinite(got).all() and ((got.double().cpu() - want).abs() <= bound).all()


def test_eviction_in_a_page_whose_heads_lie_2_gib_apart(device):
    # one page of 2^24 tokens of a 4-bit pool with head_dim 256: a head's codes are 2^31 bytes
    block, n, budget, recent = 1 << 24, 700, 300, 40
    g = torch.Generator().manual_seed(3)
    small = [torch.randint(0, 256, (1, 2, 768, w), generator=g, dtype=torch.uint8).to(device) for w in (128, 128, 8, 8)]
    weights = torch.randint(0, 9, (1, 2, 768), generator=g).float().to(device)
    big = [torch.zeros(1, 2, block, t.shape[-1], dtype=torch.uint8, device=device) for t in small]
    scores = torch.zeros(1, 2, block, device=device)
    scores[:, :, :768] = weights
    for b, t in zip(big, small):
        b[:, :, :768] = t
    lens, table = i32([n], device), i32([[0]], device)
    results = []
    for (k, v, ks, vs), w in ((small, weights), (big, scores)):
        k, v = (t.view(torch.float4_e2m1fn_x2) for t in (k, v))
        results.append(slo_attn.evict_kv(k, v, w, lens, table, budget, recent, ks, vs))
    assert torch.equal(results[0][1], results[1][1]) and results[1][0].tolist() == [budget]
    for b, t in zip([*big, scores[..., None]], [*small, weights[..., None]]):
        assert torch.equal(b[:, :, :768], t)
        assert not b[:, :, 768:1 << 16].any() and not b[:, :, -(1 << 16):].any()


def test_weights_of_many_rows_without_bounds(device):
    # 1,102 rows in tables of 41 pages: 29 workgroups a row, which go round the longest one's keys
    case = Rows("fp4", [], [(300, 2200), (1, 5)] + [(1 + i % 2, i % 7) for i in range(1100)], hq=2, hkv=1, seed=8, block=64)
    kc, _, ks, _ = case.pool.device(device)
    args, start = case.arguments(device), torch.zeros(case.blocks, 1, case.block, device=device)
    given = start.clone()
    slo_attn.accumulate_attention(case.q.to(device), kc, given, case.scale, num_kv_heads=1, k_scale=ks, **args)
    slo_attn.accumulate_attention(case.q.to(device), kc, start, case.scale, num_kv_heads=1, k_scale=ks, **without_bounds(case, device))
    assert torch.equal(given, start) and given.sum().item() == pytest.approx(2 * case.tokens, rel=1e-4)


@pytest.mark.parametrize("fmt,group", [("bf16", 3), ("fp8", 5), ("fp4", 6), ("bf16", 9), ("fp8", 11), ("fp4", 13), ("bf16", 15)])
def test_weights_of_groups_that_leave_columns_empty(device, fmt, group):
    # groups that do not divide a tile's 64 columns, and last tiles of few queries, over keys that every query sees
    case = Rows(fmt, [], [(37, 300), (1, 129), (9, 0)], hq=2 * group, hkv=2, seed=group, gain=8.0)
    kc, _, ks, _ = case.pool.device(device)
    start = torch.zeros(case.blocks, 2, case.block)
    want, bound = expected(case, start)
    got = start.to(device)
    slo_attn.accumulate_attention(case.q.to(device), kc, got, case.scale, num_kv_heads=2, k_scale=ks, **case.arguments(device))
    assert torch.isfinite(got).all() and ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("mixed", [False, True], ids=["v0", "mixed"])
@pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3fn", "fp4_e2m1"])
def test_cold_prompts_without_tables_are_weighed(device, fmt, mixed):
    # whole prompts attend to their new rows; their weights go to the pages that their slots say
    hq, hkv, block, lens = 8, 2, 64, [130, 1, 64]
    tables = [[4, 0, 7], [2, -1, -1], [5, -1, -1]]
    pool = slo_attn.KVPool(1, 9, block, hkv, D, fmt, device, track_scores=True)
    layer = slo_attn.Attention(hq, D, D ** -0.5, hkv)
    pool.attach([layer])
    pool.kv.zero_()
    pool.scores.fill_(50.0)
    g = torch.Generator().manual_seed(6)
    n = sum(lens) + mixed
    q, k, v = (random_values(g, n, h, D).to(device) for h in (hq, hkv, hkv))
    slots = [t[j // block] * block + j % block for t, m in zip(tables, lens) for j in range(m)]
    cu = i32([0, 130, 131, 195], device)
    if mixed:  # a decode row's first token beside them, in block 8
        meta = slo_attn.MixedAttentionContext(1, n - 1, i32([1], device), i32([[8]], device), cu, cu, None, 130, 130, False)
        slo_attn.set_context(False, slot_mapping=i32([8 * block] + slots, device), mixed=meta)
    else:
        slo_attn.set_context(True, cu, cu, 130, 130, i32(slots, device), None, None)
    out = layer(q, k, v)
    slo_attn.reset_context()
    got = pool.scores[0].clone()
    # the same call with the tables written out
    kc, _, ks, _ = pool.layer(0)
    want = torch.full_like(got, 50.0)
    slo_attn.accumulate_attention(q[mixed:], kc, want, D ** -0.5, num_kv_heads=hkv, k_scale=ks, num_prefill=3, prefill_cu_q=cu,
                                  prefill_cu_k=cu, max_q=130, max_k=130, prefill_tables=i32(tables, device))
    if mixed:
        want[8, :, 0] = 4.0  # the only key of the group's four heads
        got[8, :, 0] = got[8, :, 0].round(decimals=5)
    assert torch.equal(got, want)
    for t, m in zip(tables, lens):
        row = torch.stack([got[t[j // block], :, j % block] for j in range(m)])
        assert torch.allclose(row.sum(0), torch.full((hkv,), 4.0 * m, device=device), rtol=1e-4)
    alone = slo_attn.paged_attention(q[mixed:], None, None, D ** -0.5, num_kv_heads=hkv, num_prefill=3, prefill_cu_q=cu,
                                     prefill_cu_k=cu, max_q=130, max_k=130, k=k[mixed:], v=v[mixed:])
    assert torch.equal(out[mixed:], alone)


@pytest.mark.parametrize("fmt,lens,hq,hkv,width", [("bf16", [2047, 5], 2, 2, 33), ("bf16", [1983], 2, 2, 31), ("fp8", [4100, 0, 64], 4, 4, 65),
                                                   ("fp4", [8200], 1, 1, 129), ("fp4", [8000, 9], 2, 1, 126)])
def test_few_long_decode_rows(device, fmt, lens, hq, hkv, width):
    case = Rows(fmt, lens, hq=hq, hkv=hkv, seed=width, gain=3.0, spare=width - max(-(-n // 64) for n in lens))
    kc, _, ks, _ = case.pool.device(device)
    start = torch.rand(case.blocks, hkv, case.block, generator=torch.Generator().manual_seed(2))
    want, bound = expected(case, start)
    got = start.to(device)
    slo_attn.accumulate_attention(case.q.to(device), kc, got, case.scale, num_kv_heads=hkv, k_scale=ks, **case.arguments(device))
    assert torch.isfinite(got).all() and ((got.double().cpu() - want).abs() <= bound).all()


def test_captured_cold_prompts_are_weighed_on_every_replay(device):
    # the pages come from the slots inside the graph: a replay goes where the slots then say
    hq, hkv, block, lens = 8, 2, 64, [70, 33]
    pool = slo_attn.KVPool(1, 6, block, hkv, D, "bf16", device, track_scores=True)
    layer = slo_attn.Attention(hq, D, D ** -0.5, hkv)
    pool.attach([layer])
    pool.kv.zero_()
    g = torch.Generator().manual_seed(9)
    q, k, v = (random_values(g, sum(lens), h, D).to(device) for h in (hq, hkv, hkv))
    cu, slots = i32([0, 70, 103], device), torch.full((sum(lens),), -1, dtype=torch.int32, device=device)

    def step():
        slo_attn.set_context(True, cu, cu, 70, 70, slots, None, None)
        try:
            return layer(q, k, v)
        finally:
            slo_attn.reset_context()

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for tables in ([[0, 3], [5]], [[4, 1], [2]], [[0, 3], [5]]):
        slots.copy_(i32([t[j // block] * block + j % block for t, n in zip(tables, lens) for j in range(n)], device))
        pool.scores.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone(), pool.scores.clone()
        pool.scores.fill_(9.0)
        want = step()
        assert torch.equal(got[0], want) and torch.equal(got[1], pool.scores)
        live = torch.zeros_like(got[1], dtype=torch.bool)
        for t, n in zip(tables, lens):
            for j in range(n):
                live[0, t[j // block], :, j % block] = True
        assert (got[1][~live] == 9).all() and got[1][live].sum().item() == pytest.approx(hq * sum(lens), rel=1e-4)
