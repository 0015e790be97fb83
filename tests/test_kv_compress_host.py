"""The 4-bit pool and eviction on the CPU: the definition against brute force,
the C-ABI's refusals, and KVPool's shapes and lifecycle."""
import ctypes

import numpy as np
import pytest
import torch

import slo_attn
from oracle import fp4 as ofp4
from oracle import kv_scores
from slo_attn import KVPool, _lib, kv_block_bytes


def test_definition_codes_are_the_nearest_values():
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((50, 64)) * np.exp(3 * rng.standard_normal((50, 1)))).to(torch.bfloat16)
    codes, scale = ofp4.quantize_kv(x.float().numpy())
    back = ofp4.dequantize_kv(codes, scale)
    xd = x.double().numpy().reshape(50, 2, 32)
    s = np.exp2(scale.astype(np.float64) - 127)
    assert (np.abs(xd).max(-1) < 7 * s).all() and (np.abs(xd).max(-1) >= 3.5 * s).all()
    grid = np.concatenate((ofp4.VALUES, -ofp4.VALUES))
    nearest = np.abs(xd[..., None] - grid * s[..., None, None]).min(-1)
    assert np.array_equal(np.abs(xd - back.reshape(50, 2, 32)), nearest)
    # ties to the even code, saturation, zeros keep their sign
    t = np.zeros((1, 32), dtype=np.float32)
    t[0, :9] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.75, -0.0]
    codes, scale = ofp4.quantize_kv(t)
    assert scale[0, 0] == 127
    assert ofp4.dequantize_kv(codes, scale)[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6] and codes[0, 4] == 8
    big = np.full((1, 32), np.inf, dtype=np.float32)
    assert np.isfinite(ofp4.dequantize_kv(*ofp4.quantize_kv(big))).all()
    assert (ofp4.quantize_kv(np.zeros((1, 32), np.float32))[1] == 63).all()


def test_definition_of_the_choice():
    nan, inf = float("nan"), float("inf")
    assert kv_scores.choose(np.array([1.0, 5, 5, 2, 0, 9]), 3, 1) == [1, 2, 5]
    assert kv_scores.choose(np.array([1.0, 1, 1, 1]), 2, 0) == [0, 1]
    assert kv_scores.choose(np.array([nan, -inf, 0.0, inf, nan]), 3, 1) == [2, 3, 4]
    assert kv_scores.choose(np.array([1.0, 2, 3]), 2, 2) == [1, 2]
    assert kv_scores.choose(np.array([1.0, 2]), 5, 1) == [0, 1]


def test_block_bytes_and_pool_shapes():
    assert kv_block_bytes(36, 256, 8, 128, "fp4_e2m1") == 36 * 256 * 8 * 136
    assert kv_block_bytes(2, 64, 4, 128, "bf16", track_scores=True) == kv_block_bytes(2, 64, 4, 128) + 4 * 2 * 64 * 4
    pool = KVPool(2, 5, 64, 4, 128, "fp4_e2m1", track_scores=True)
    assert pool.kv.shape == (2, 2, 5, 4, 64, 64) and pool.scale.shape == (2, 2, 5, 4, 64, 4)
    total = pool.kv.numel() + pool.scale.numel() + 4 * pool.scores.numel()
    assert total == 5 * kv_block_bytes(2, 64, 4, 128, "fp4_e2m1", True)
    k, v, ks, vs = pool.layer(1)
    assert k.dtype == torch.float4_e2m1fn_x2 and k.shape == (5, 4, 64, 64) and k.data_ptr() == pool.kv[0, 1].data_ptr()
    assert vs.data_ptr() == pool.scale[1, 1].data_ptr() and not pool.fp8
    assert pool.scores.shape == (2, 5, 4, 64)
    with pytest.raises(ValueError):
        KVPool(1, 1, 64, 1, 48, "fp4_e2m1")


@pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3fn", "fp4_e2m1"])
def test_blocks_move_with_scales_and_scores(fmt):
    pool = KVPool(2, 6, 64, 2, 128, fmt, track_scores=True)
    g = torch.Generator().manual_seed(1)

    def fill():
        pool.kv.copy_(torch.randint(0, 50, pool.kv.shape, generator=g))
        if pool.scale is not None:
            pool.scale.copy_(torch.randint(1, 50, pool.scale.shape, generator=g))
        pool.scores.copy_(torch.rand(pool.scores.shape, generator=g))

    fill()
    pool.copy_blocks([1, 4], [0, 5])
    parts = [pool.kv, pool.scores.unsqueeze(0)] + ([pool.scale] if pool.scale is not None else [])
    for t in parts:
        assert torch.equal(t[:, :, 0], t[:, :, 1]) and torch.equal(t[:, :, 5], t[:, :, 4])
    image = pool.snapshot([1, 3])
    saved = [t.clone() for t in parts]
    fill()
    pool.restore(image)
    for t, old in zip(parts, saved):
        assert torch.equal(t[:, :, [1, 3]], old[:, :, [1, 3]])
    pool.reset_blocks([3])
    assert not pool.scores[:, 3].any() and not pool.kv[:, :, 3].any()
    if fmt == "fp4_e2m1":
        assert (pool.scale[:, :, 3] == 127).all()  # a scale of 1


def test_attach_sets_scores():
    pool = KVPool(2, 3, 64, 2, 128, "fp4_e2m1", track_scores=True)
    layers = [slo_attn.Attention(4, 128, 0.1, 2) for _ in range(2)]
    assert pool.attach(layers) == 2
    assert layers[1].kv_scores.data_ptr() == pool.scores[1].data_ptr()
    assert layers[1].k_scale.data_ptr() == pool.scale[0, 1].data_ptr()
    KVPool(2, 3, 64, 2, 128).attach(layers)
    assert layers[0].kv_scores is None and layers[0].k_scale is None


def attention_args(**over):
    a = _lib.PagedAttentionArgs()
    a.head_dim, a.num_heads, a.num_kv_heads, a.softmax_scale, a.kv_dtype = 128, 32, 8, 0.1, _lib.KV_FP4_E2M1
    a.q = a.out = a.k_cache = a.v_cache = a.k_scale = a.v_scale = 4096
    a.q_row_stride = a.out_row_stride = 32 * 128
    a.num_q_rows = a.num_decode = 4
    a.num_blocks, a.block_size, a.phases = 2, 256, 3
    a.decode_lens, a.decode_tables, a.decode_table_stride, a.decode_table_width = 4096, 4096, 16, 16
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("over,code,word", [
    (dict(head_dim=64), 4, "head_dim"), (dict(num_heads=30), 1, "multiple"), (dict(num_heads=136), 4, "16 query heads"),
    (dict(num_decode=5), 1, "row counts"), (dict(num_decode=-1), 1, "row counts"), (dict(softmax_scale=0.0), 1, "softmax_scale"),
    (dict(softmax_scale=float("inf")), 1, "softmax_scale"), (dict(q=0), 1, "null"), (dict(q=4104), 1, "aligned"),
    (dict(q_row_stride=4100), 1, "aligned"), (dict(k_cache=0), 1, "pool"), (dict(k_scale=0), 1, "scale"),
    (dict(block_size=96), 4, "block_size"), (dict(decode_lens=0), 1, "metadata"), (dict(decode_table_width=0), 1, "metadata"),
    (dict(num_prefill=1, max_q=3), 1, "metadata"), (dict(decode_table_width=1 << 23), 4, "tokens"),
    (dict(num_decode=40000, num_q_rows=40000), 4, "rows"), (dict(num_prefill=40000), 4, "rows"),
])
def test_attention_refusals_without_a_gpu(over, code, word):
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    for call in (lambda a: lib.slo_paged_attention_fp4(bytes(a), None),
                 lambda a: lib.slo_paged_attention_fp4_workspace_bytes(bytes(a), ctypes.byref(need)),
                 lambda a: lib.slo_accumulate_attention(bytes(a), 4096, None),
                 lambda a: lib.slo_accumulate_attention_workspace_bytes(bytes(a), ctypes.byref(need))):
        assert call(attention_args(**over)) == code
        assert word in lib.slo_last_error().decode()


def test_workspace_refusals_without_a_gpu():
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    a = attention_args(decode_table_width=64)
    assert lib.slo_accumulate_attention_workspace_bytes(bytes(a), ctypes.byref(need)) == 0 and need.value > 0
    a.workspace, a.workspace_bytes = 4096, need.value - 1
    assert lib.slo_accumulate_attention(bytes(a), 4096, None) == 3
    a.workspace, a.workspace_bytes = None, need.value
    assert lib.slo_accumulate_attention(bytes(a), 4096, None) == 3
    assert lib.slo_accumulate_attention(bytes(attention_args(kv_dtype=3)), 4096, None) == 1
    assert lib.slo_paged_attention_fp4(bytes(attention_args(kv_dtype=1)), None) == 1
    assert lib.slo_paged_attention_fp4(bytes(attention_args(store_slot_mapping=4096)), None) == 1
    a = attention_args(decode_table_width=4096, num_decode=1)  # one long row: split, so it needs a workspace
    assert lib.slo_paged_attention_fp4_workspace_bytes(bytes(a), ctypes.byref(need)) == 0 and need.value > 0
    assert lib.slo_paged_attention_fp4(bytes(a), None) == 3
    # nothing to do
    assert lib.slo_paged_attention_fp4(bytes(attention_args(num_decode=0)), None) == 0
    assert lib.slo_accumulate_attention(bytes(attention_args(num_decode=0)), 4096, None) == 0
    assert lib.slo_paged_attention_fp4(None, None) == 1 and lib.slo_accumulate_attention(None, None, None) == 1


def test_pool_entry_refusals_without_a_gpu():
    lib = _lib.load()

    def store(n=4, heads=8, d=128, key=4096, stride=1024, blocks=2, floor=2.0 ** -64, scale=4096):
        return lib.slo_store_kvcache_fp4(key, stride, 4096, 1024, 4096, n, heads, d, 4096, 4096, scale, 4096, blocks, 256, floor, None)

    assert store(n=0) == 0 and store(n=-1) == 1 and store(d=96) == 4 and store(key=4104) == 1 and store(stride=1020) == 1
    assert store(blocks=0) == 1 and store(scale=None) == 1 and store(floor=0.3) == 1 and store(floor=-1.0) == 1
    assert store(floor=0.0) == 1 and store(heads=0) == 1

    def load(kv=2, n=4, d=128, scale=4096, out=4096, blocks=2):
        return lib.slo_load_kvcache(4096, 4096, scale, 4096, kv, blocks, 256, 4096, n, 8, d, out, 4096, None)

    assert load(n=0) == 0 and load(n=-1) == 1 and load(kv=3) == 1 and load(d=96) == 4 and load(scale=None) == 1
    assert load(out=None) == 1 and load(out=4104) == 1 and load(blocks=0) == 1


def test_evict_refusals_without_a_gpu():
    lib = _lib.load()

    def call(**over):
        a = _lib.EvictKvArgs(4096, 4096, 4096, 4096, 4096, 2, 1, 4, 256, 8, 128, 2, 4096, 4096, 4, 4, 100, 10, 4096, 4096)
        for name, value in over.items():
            setattr(a, name, value)
        return lib.slo_evict_kv(ctypes.byref(a), None)

    assert lib.slo_evict_kv(None, None) == 1 and call(num_rows=0) == 0
    for over in (dict(budget=0), dict(recent=101), dict(recent=-1), dict(num_layers=0), dict(kv_dtype=3), dict(num_blocks=0),
                 dict(k_scale=None), dict(scores=None), dict(kept=None), dict(k_cache=4104), dict(table_width=0),
                 dict(scores=4100)):
        assert call(**over) == 1, over
    for over in (dict(head_dim=96), dict(num_rows=65536), dict(table_width=1 << 20), dict(block_size=96)):
        assert call(**over) == 4, over


def test_packed_arguments_are_the_struct():
    values = {t: i for i, t in enumerate(_lib.PagedAttentionArgs._fields_, 1)}
    a = _lib.PagedAttentionArgs()
    for (name, _), i in values.items():
        setattr(a, name, i)
    packed = _lib.pack_attention_args(*range(1, len(values) + 1))
    assert len(packed) == ctypes.sizeof(a)
    back = _lib.PagedAttentionArgs.from_buffer_copy(packed)
    for name, _ in _lib.PagedAttentionArgs._fields_:
        assert getattr(back, name) == getattr(a, name), name


def test_host_layer_refuses_cpu_tensors():
    pool = KVPool(1, 2, 64, 2, 128, "fp4_e2m1", track_scores=True)
    k, v, ks, vs = pool.layer(0)
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(2, dtype=torch.int32)
    calls = (lambda: slo_attn.store_kvcache(x, x, k, v, slots, ks, vs), lambda: slo_attn.load_kvcache(k, v, slots, ks, vs),
             lambda: slo_attn.accumulate_attention(x, k, pool.scores[0], 0.1, num_kv_heads=2, k_scale=ks),
             lambda: pool.evict(slots, slots.view(2, 1), 3, 1), lambda: pool.read(0, slots))
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
