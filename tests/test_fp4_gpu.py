"""The 4-bit KV pool on the GPU: write, read back and paged attention against
the 64-bit definition (oracle/fp4.py, oracle/kv_scores.py)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import slo_attn
from fp4_cases import D, STALE, Pool, Rows, i32, random_values
from oracle import fp4 as ofp4
from oracle import fp8 as ofp8

pytestmark = pytest.mark.gpu


def fp4(t):
    return t.view(torch.float4_e2m1fn_x2)


def store(k, v, slots, blocks, block, device, floor=2.0 ** -64, kd=None, vd=None):
    hkv, d = k.shape[1], k.shape[2]
    pages = [torch.full((blocks, hkv, block, d // 2), 0xA5, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.full((blocks, hkv, block, d // 32), STALE, dtype=torch.uint8, device=device) for _ in range(2)]
    slo_attn.store_kvcache(k.to(device) if kd is None else kd, v.to(device) if vd is None else vd, fp4(pages[0]),
                           fp4(pages[1]), i32(slots, device), scales[0], scales[1], floor)
    return pages, scales


def check_store(k, v, slots, blocks, block, pages, scales, floor=2.0 ** -64):
    want_p = [np.full(tuple(p.shape), 0xA5, dtype=np.uint8) for p in pages]
    want_s = [np.full(tuple(s.shape), STALE, dtype=np.uint8) for s in scales]
    ofp4.store_kvcache(k.float().numpy(), v.float().numpy(), *want_p, *want_s, slots, floor)
    for got, want in zip(pages + scales, want_p + want_s):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("anchor", [0.0, 6.0, 6.96875, 7.0, 2.0 ** -70, 3.0e38])
def test_every_bf16_value_has_the_definitions_code(device, anchor):
    # one value and an anchor that sets the scale in every group of 32; every other value twice
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536, 32, dtype=torch.bfloat16)
    x[:, 5] = bits
    x[:, 18] = bits.flip(0) if anchor == 0.0 else anchor
    x = x.view(4096, 4, 128)
    slots = list(range(4096))
    pages, scales = store(x, x.neg(), slots, 16, 256, device)
    check_store(x, x.neg(), slots, 16, 256, pages, scales)


@pytest.mark.parametrize("d,hkv,n,block", [(64, 1, 5, 64), (128, 8, 37, 256), (256, 3, 9, 192), (128, 2, 1, 64)])
def test_store_of_views_skips_slots_outside_the_pool(device, d, hkv, n, block):
    g = torch.Generator().manual_seed(d + n)
    qkv = random_values(g, n, hkv * 2 + 3, d)
    k, v = qkv[:, 3:3 + hkv], qkv[:, 3 + hkv:]
    blocks = 3
    slots = torch.randperm(blocks * block, generator=g)[:n].tolist()
    slots[0] = -1
    if n > 2:
        slots[1], slots[2] = blocks * block, -7
    dev = qkv.to(device)
    pages, scales = store(k, v, slots, blocks, block, device, 2.0 ** -20, dev[:, 3:3 + hkv], dev[:, 3 + hkv:])
    check_store(k, v, slots, blocks, block, pages, scales, 2.0 ** -20)


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_load_reads_back_what_is_stored(device, fmt):
    g = torch.Generator().manual_seed(3)
    pool = Pool(fmt, 5, 64, 2)
    table = [4, 0, 2]
    pool.write(table, random_values(g, 150, 2, D), random_values(g, 150, 2, D))
    kc, vc, ks, vs = pool.device(device)
    place = torch.randperm(150, generator=g)[:77].tolist()
    slots = [table[j // 64] * 64 + j % 64 for j in place] + [-1, 5 * 64, -400]
    got = slo_attn.load_kvcache(kc, vc, i32(slots, device), ks, vs)
    for side in (0, 1):
        want = pool.values(table, 150, side)[0][place]
        if fmt == "fp8":  # one rounding of code * scale in fp32, one to bf16
            assert ((got[side][:77].double().cpu() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -24)).all()
        else:
            assert torch.equal(got[side][:77].double().cpu(), want)
        assert not got[side][77:].any()
    assert slo_attn.load_kvcache(kc, vc, i32([], device), ks, vs)[0].shape == (0, 2, D)


CASES = {
    "one_key": dict(lens=[1]),
    "empty_rows": dict(lens=[0, 1, 0, 31, 32, 33, 63, 64, 65, 0]),
    "odd_lengths": dict(lens=[127, 128, 129, 255, 257, 500], hq=16, hkv=4, block=128),
    "split_rows": dict(lens=[3000, 17, 1023, 2049], hq=8, hkv=2, gain=2.0),
    "group_1": dict(lens=[70, 200], hq=2, hkv=2, block=192),
    "group_5": dict(lens=[70, 300], hq=10, hkv=2, gain=3.0),
    "group_7_prefill": dict(lens=[90], chunks=[(37, 0), (5, 100), (1, 0)], hq=28, hkv=4),
    "group_16": dict(lens=[333], chunks=[(20, 45)], hq=16, hkv=1, block=256),
    "peaked": dict(lens=[400, 900], chunks=[(70, 130)], hq=8, hkv=2, gain=30.0),
    "chunks": dict(lens=[], chunks=[(64, 0), (33, 64), (130, 701), (1, 511), (3, 0)], hq=16, hkv=4),
    "fewer_keys_than_queries": dict(lens=[], chunks=[(40, -7), (20, -20), (9, 3)], hq=8, hkv=2),
    "long_prefix": dict(lens=[], chunks=[(3, 2600)], hq=8, hkv=2),
    "mixed": dict(lens=[5, 700, 64], chunks=[(100, 0), (50, 333)], block=256),
    "negative_scale": dict(lens=[80], chunks=[(30, 20)], hq=8, hkv=2, scale=-0.11),
    "rows_past_lds": dict(lens=[4500, 1, 1025, 0, 5000], hq=8, hkv=2, block=256, gain=4.0),
    "rows_past_lds_group_16": dict(lens=[1500, 1030, 33], hq=16, hkv=1, block=64),
    "many_rows": dict(lens=[(37 * i) % 130 for i in range(150)], chunks=[(i % 5, 3 * i) for i in range(70)], hq=4, hkv=2),
    "many_tiles": dict(lens=[], chunks=[(2300, 30), (40, 0)], hq=16, hkv=1),
    "tables_far_wider_than_the_rows": dict(lens=[100, 5, 0], chunks=[(9, 70), (2, 0)], hq=8, hkv=2, spare=90),
    "pages_not_in_the_pool": dict(lens=[200, 60], chunks=[(20, 140)], hq=8, hkv=2, holes=[(0, 1, -1), (1, 0, 10 ** 6), (2, 0, -5)]),
}


@pytest.mark.parametrize("name", CASES)
def test_attention_over_a_4_bit_pool(device, name):
    case = Rows("fp4", **{"seed": len(name), **CASES[name]})
    kc, vc, ks, vs = case.pool.device(device)
    got = slo_attn.paged_attention(case.q.to(device), kc, vc, case.scale, num_kv_heads=case.hkv, k_scale=ks, v_scale=vs,
                                   **case.arguments(device))
    want, _, bound = case.attend()
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), f"{(off / bound).max():.3f} of the bound"


def test_attention_of_views_into_a_wider_output(device):
    case = Rows("fp4", [100, 30], [(17, 40)], hq=8, hkv=2, seed=4)
    kc, vc, ks, vs = case.pool.device(device)
    wide = torch.zeros(case.tokens, 12, D, dtype=torch.bfloat16, device=device)
    wide[:, :8] = case.q.to(device)
    out = torch.full((case.tokens + 2, 10, D), 7.0, dtype=torch.bfloat16, device=device)
    args = dict(num_kv_heads=2, k_scale=ks.view(torch.float8_e8m0fnu), v_scale=vs, **case.arguments(device))
    got = slo_attn.paged_attention(wide[:, :8], kc, vc, case.scale, out=out[:case.tokens, :8], **args)
    assert got.data_ptr() == out.data_ptr()
    plain = slo_attn.paged_attention(case.q.to(device), kc, vc, case.scale, **args)
    assert torch.equal(out[:case.tokens, :8], plain)
    assert (out[case.tokens:] == 7).all() and (out[:, 8:] == 7).all()
    # one phase at a time: the other's rows stay as they are
    for phases, mine in ((slo_attn._lib.PHASE_DECODE, slice(0, 2)), (slo_attn._lib.PHASE_PREFILL, slice(2, None))):
        o = torch.full_like(plain, 5.0)
        slo_attn.paged_attention(case.q.to(device), kc, vc, case.scale, out=o, phases=phases, **args)
        other = torch.ones(case.tokens, dtype=torch.bool)
        other[mine] = False
        assert torch.equal(o[mine], plain[mine]) and (o[other.to(device)] == 5).all()


def test_rows_past_every_row_get_zeros_and_bounds_may_be_capacities(device):
    case = Rows("fp4", [100, 30], [(17, 40), (5, 0)], hq=8, hkv=2, seed=4)
    kc, vc, ks, vs = case.pool.device(device)
    args = dict(num_kv_heads=2, k_scale=ks, v_scale=vs, **case.arguments(device))
    q = torch.cat((case.q, torch.full((40, 8, D), float("nan"), dtype=torch.bfloat16))).to(device)
    want, _, bound = case.attend()
    args["max_q"], args["max_k"] = 60, 5000
    for phases in (1, 2, 3):
        out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device=device)
        slo_attn.paged_attention(q, kc, vc, case.scale, out=out, phases=phases, **args)
        assert not out[case.tokens:].any()
        for bit, rows in ((1, slice(0, 2)), (2, slice(2, case.tokens))):
            if phases & bit:
                assert ((out[rows].double().cpu() - want[rows]).abs() <= bound[rows]).all()
            else:
                assert (out[rows] == 3).all()
    decode = {k: v for k, v in args.items() if "prefill" not in k and "max" not in k}
    out = slo_attn.paged_attention(q[:5], kc, vc, case.scale, out=torch.ones_like(q[:5]), **decode)
    assert not out[2:].any() and out[:2].any()


def test_captured_mixed_steps_on_a_4_bit_pool(device):
    # a bucket's graph (metadata, store, attention, weights) against the same bucket run eagerly
    hq, hkv, block, width = 8, 2, 64, 4
    pool = slo_attn.KVPool(2, 24, block, hkv, D, "fp4_e2m1", device, track_scores=True)
    layers = [slo_attn.Attention(hq, D, D ** -0.5, hkv) for _ in range(2)]
    pool.attach(layers)
    g = torch.Generator().manual_seed(3)
    table = random_values(g, 50, hq + 2 * hkv, D).to(device)

    def forward(ids, positions):
        x = table[ids]
        out = 0
        for layer in layers:
            out = out + layer(x[:, :hq].contiguous(), x[:, hq:hq + hkv], x[:, hq + hkv:])
        return out

    buf = slo_attn.MixedStepBuffers(4, 3, 120, width, block, width * block, device)
    graph = slo_attn.MixedStepGraph(buf, forward)
    pool.kv.zero_(), pool.scale.fill_(127), pool.scores.zero_()
    steps = [([], [(0, 60), (0, 33)], [[0, 1], [2]], list(range(40)) + list(range(50)) + [7, 8, 9]),
             ([60, 33], [(0, 20)], [[0, 1], [2], [5]], list(range(22))),
             ([61, 34, 20], [(0, 1)], [[0, 1], [2], [5], [6]], [1, 2, 3, 4])]
    for step in steps:
        before = pool.kv.clone(), pool.scale.clone(), pool.scores.clone()
        got = graph.run(*step).clone()
        torch.cuda.synchronize()
        after = pool.kv.clone(), pool.scale.clone(), pool.scores.clone()
        for t, b in zip((pool.kv, pool.scale, pool.scores), before):
            t.copy_(b)
        buf.build()
        buf.set_context(True)
        want = forward(buf.input_ids, buf.positions)
        slo_attn.reset_context()
        assert torch.isfinite(want).all() and torch.equal(got, want)
        assert all(torch.equal(x, y) for x, y in zip(after, (pool.kv, pool.scale, pool.scores)))
    assert pool.scores.any()


def test_pool_past_4_gib(device):
    # the last blocks of a pool whose codes pass 2^32 bytes and scales 2^28
    blocks, block, hkv = 33000, 256, 8
    case = Rows("fp4", [300, 40], [(10, 100)], hq=16, hkv=hkv, block=block, seed=9)
    kc, vc, ks, vs = case.pool.device(device)
    big = [torch.zeros(blocks, hkv, block, w, dtype=torch.uint8, device=device) for w in (64, 64, 4, 4)]
    for b, t in zip(big, (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)):
        b[-case.blocks:] = t
    shift = blocks - case.blocks
    case.tables = [[p + shift if p >= 0 else p for p in t] for t in case.tables]
    args = case.arguments(device)
    got = slo_attn.paged_attention(case.q.to(device), fp4(big[0]), fp4(big[1]), case.scale, num_kv_heads=hkv,
                                   k_scale=big[2], v_scale=big[3], **args)
    case.tables = [[p - shift if p >= 0 else p for p in t] for t in case.tables]
    small = slo_attn.paged_attention(case.q.to(device), kc, vc, case.scale, num_kv_heads=hkv, k_scale=ks, v_scale=vs,
                                     **case.arguments(device))
    assert torch.equal(got, small)
    scores = torch.zeros(blocks, hkv, block, device=device)
    slo_attn.accumulate_attention(case.q.to(device), fp4(big[0]), scores, case.scale, num_kv_heads=hkv, k_scale=big[2], **args)
    few = torch.zeros(case.blocks, hkv, block, device=device)
    slo_attn.accumulate_attention(case.q.to(device), kc, few, case.scale, num_kv_heads=hkv, k_scale=ks,
                                  **case.arguments(device))
    assert torch.equal(scores[shift:], few) and not scores[:shift].any()


def test_cold_prefill_rows_read_the_new_rows(device):
    # prefill rows without tables read K/V as given, beside decode rows of the 4-bit pool
    case = Rows("fp4", [70, 5], [(33, 0), (50, 0)], hq=16, hkv=4, seed=5)
    kc, vc, ks, vs = case.pool.device(device)
    args = case.arguments(device)
    args["prefill_tables"] = None
    g = torch.Generator().manual_seed(1)
    k, v = (random_values(g, 83, 4, D).to(device) for _ in range(2))
    q = case.q.to(device)
    got = slo_attn.paged_attention(q, kc, vc, case.scale, num_kv_heads=4, k_scale=ks, v_scale=vs, k=k, v=v, **args)
    alone = slo_attn.paged_attention(q[2:], None, None, case.scale, num_kv_heads=4, num_prefill=2,
                                     prefill_cu_q=args["prefill_cu_q"], prefill_cu_k=args["prefill_cu_k"], max_q=50,
                                     max_k=50, k=k, v=v)
    want, _, bound = case.attend()
    assert torch.equal(got[2:], alone)
    assert ((got[:2].double().cpu() - want[:2]).abs() <= bound[:2]).all()


def test_step_through_the_attention_layer(device):
    # forward_mixed and Attention.forward over a 4-bit KVPool: the store, then the launch
    hq, hkv, block = 16, 4, 64
    pool = slo_attn.KVPool(2, 12, block, hkv, D, "fp4_e2m1", device, track_scores=True)
    layers = [slo_attn.Attention(hq, D, D ** -0.5, hkv) for _ in range(2)]
    assert pool.attach(layers) == 2
    g = torch.Generator().manual_seed(8)
    n = 70 + 30
    q = random_values(g, n, hq, D).to(device)
    qkv = random_values(g, n, 2 * hkv, D).to(device)
    k, v = qkv[:, :hkv], qkv[:, hkv:]
    tables = [[3, 7, -1], [1, -1, -1]]
    slots = [tables[0][j // block] * block + j % block for j in range(70)] + [block + j for j in range(30)]
    meta = slo_attn.MixedAttentionContext(0, n, None, None, i32([0, 70, 100], device), i32([0, 70, 100], device),
                                          i32(tables, device), 70, 70, True)
    slo_attn.set_context(True, slot_mapping=i32(slots, device))
    slo_attn.get_context().mixed = meta
    out = layers[1](q, k, v)
    kc, vc, ks, vs = pool.layer(1)
    want = [t.clone() for t in (pool.kv[:, 1], pool.scale[:, 1])]
    assert torch.equal(layers[1](q, k, v, kv_stored=True), out)
    assert torch.equal(pool.kv[:, 1], want[0]) and torch.equal(pool.scale[:, 1], want[1])
    assert not pool.kv[:, 0].any()
    # the fused step before attention writes the same pool bytes as a store of its k and v
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    flat = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1)
    table = slo_attn.rope_cos_sin(D, 128, 1e4, device)
    pos = torch.arange(n, device=device)
    other = slo_attn.KVPool(1, 12, block, hkv, D, "fp4_e2m1", device)
    oc = other.layer(0)
    _, k2, v2 = slo_attn.qk_norm_rope_store(flat, pos, w, w, 1e-6, table, hq, hkv, oc[0], oc[1], i32(slots, device), oc[2], oc[3])
    again = slo_attn.KVPool(1, 12, block, hkv, D, "fp4_e2m1", device)
    ac = again.layer(0)
    slo_attn.store_kvcache(k2, v2, ac[0], ac[1], i32(slots, device), ac[2], ac[3])
    assert torch.equal(other.kv, again.kv) and torch.equal(other.scale, again.scale) and other.kv.any()
    # V0 decode of the first row's last token, from the pool alone
    slo_attn.set_context(False, slot_mapping=i32([slots[69]], device), context_lens=i32([70], device),
                         block_tables=i32(tables[:1], device))
    o = layers[1](q[69:70], k[69:70], v[69:70])
    slo_attn.reset_context()
    assert o.shape == (1, 1, hq, D)
    kk, vv = pool.read(1, i32(slots[:70], device))
    assert torch.equal(kk.float(), torch.from_numpy(ofp4.dequantize_kv(*ofp4.quantize_kv(k[:70].float().cpu().numpy()))).float().to(device))
    # each of the two is within 2^-8 (sum w|v| + 2 |out|) of the exact output
    assert (o[0, 0].float() - out[69].float()).abs().max() <= 6 * 2.0 ** -8 * vv.float().abs().max()


def test_captured_decode_replays(device):
    case = Rows("fp4", [1500, 40, 700], hq=16, hkv=4, seed=11)
    kc, vc, ks, vs = case.pool.device(device)
    args = case.arguments(device)
    q = case.q.to(device)
    scores = torch.zeros(case.blocks, 4, case.block, device=device)

    def step():
        out = slo_attn.paged_attention(q, kc, vc, case.scale, num_kv_heads=4, k_scale=ks, v_scale=vs, **args)
        slo_attn.accumulate_attention(q, kc, scores, case.scale, num_kv_heads=4, k_scale=ks, **args)
        return out

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for lens in ([1500, 40, 700], [1, 0, 699], [777, 33, 64], [1500, 40, 700]):
        args["decode_lens"].copy_(i32(lens, device))
        scores.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone(), scores.clone()
        scores.zero_()
        want = step()
        assert torch.equal(got[0], want) and torch.equal(got[1], scores)


def test_two_streams_at_once(device):
    cases = [Rows("fp4", [2500, 300], [(60, 900)], hq=16, hkv=4, seed=s) for s in (21, 22)]
    states = [(c.q.to(device), c.pool.device(device), c.arguments(device)) for c in cases]

    def run(i):
        q, (kc, vc, ks, vs), args = states[i]
        s = torch.zeros(cases[i].blocks, 4, cases[i].block, device=device)
        slo_attn.accumulate_attention(q, kc, s, cases[i].scale, num_kv_heads=4, k_scale=ks, **args)
        return slo_attn.paged_attention(q, kc, vc, cases[i].scale, num_kv_heads=4, k_scale=ks, v_scale=vs, **args), s

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = run(i)
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])


def test_refusals(device):
    case = Rows("fp4", [40], [(3, 10)], hq=8, hkv=2)
    kc, vc, ks, vs = case.pool.device(device)
    q, args = case.q.to(device), case.arguments(device)

    def call(kc=kc, vc=vc, ks=ks, vs=vs, q=q, scale=0.1, hkv=2, **over):
        return slo_attn.paged_attention(q, kc, vc, scale, num_kv_heads=hkv, k_scale=ks, v_scale=vs, **{**args, **over})

    for error, over in ((ValueError, dict(ks=None)), (ValueError, dict(vs=ks.float())), (ValueError, dict(hkv=4)),
                        (ValueError, dict(noalloc=True)), (TypeError, dict(q=q.float())), (RuntimeError, dict(scale=0.0)),
                        (RuntimeError, dict(scale=float("nan"))), (ValueError, dict(ks=ks[:, :, :32])),
                        (TypeError, dict(vc=vc.view(torch.uint8))), (ValueError, dict(num_decode=5)),
                        (ValueError, dict(decode_tables=args["decode_tables"].T)),
                        (TypeError, dict(out=torch.empty(4, 8, D, device=device)))):
        with pytest.raises(error):
            call(**over)
    k = torch.zeros(2, 2, D, dtype=torch.bfloat16, device=device)
    for floor in (0.0, 3.0, -1.0, 2.0 ** -120, float("inf")):
        with pytest.raises(RuntimeError, match="scale_floor"):
            slo_attn.store_kvcache(k, k, kc, vc, i32([0, 1], device), ks, vs, floor)
    with pytest.raises(ValueError):
        slo_attn.store_kvcache(k[:, :1], k[:, :1], kc, vc, i32([0, 1], device), ks, vs)
    with pytest.raises(ValueError):
        slo_attn.load_kvcache(kc, vc, i32([0], device))
