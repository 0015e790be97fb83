"""Window attention and the rotary layouts on the CPU: the definition by brute
force, scaled tables, given back pages, and the C-ABI's refusals."""
import ctypes
import glob
import math
import os
import re
import textwrap
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import slo_attn
from oracle import kv_scores
from oracle import window as owin
from slo_attn import _lib, window_blocks


def test_definition_of_the_window():
    for n, m, prefix, window, sinks in ((5, 12, 7, 3, 2), (4, 4, 0, 2, 0), (3, 2, -1, 4, 9), (1, 9, 8, 1, 1), (6, 6, 0, 100, 3)):
        mask = owin.visible(n, m, prefix, window, sinks)
        for i in range(n):
            for j in range(m):
                t = prefix + i
                assert mask[i, j] == (j <= t and (t - j < window or j < sinks))
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((4, 4, 8), (9, 2, 8), (9, 2, 8)))
    want = kv_scores.attend(q, k, v, 5, 0.3)[0]
    assert torch.allclose(owin.attend(q, k, v, 5, 0.3, 9, 0)[0], want, atol=1e-13)
    assert torch.allclose(owin.attend(q, k, v, 5, 0.3, 1, 9)[0], want, atol=1e-13)
    assert not owin.attend(q, k, v, -3, 0.3, 2, 1)[0][:3].any()


@pytest.mark.parametrize("window,sinks,block", [(1, 0, 64), (64, 0, 64), (65, 1, 64), (100, 64, 64), (100, 65, 64), (7, 300, 128)])
def test_blocks_that_no_later_token_sees(window, sinks, block):
    for length in (0, 1, 63, 64, 65, 128, 129, 500, 777):
        later = owin.visible(1, length, length, window, sinks)[0] if length else torch.zeros(0, dtype=torch.bool)
        whole = [b for b in range(length // block) if not later[b * block:(b + 1) * block].any()]
        assert list(window_blocks(length, window, sinks, block)) == whole
    for bad in ((0, 0, 64), (5, -1, 64), (5, 0, 0)):
        with pytest.raises(ValueError):
            window_blocks(10, *bad)


class Sequence(SimpleNamespace):
    def __len__(self):
        return self.num_tokens


@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("spans", [[(64, 0)], [(100, 4), (33, 70)], [(1, 1)], [(256, 0), (300, 2), (7, 130)]])
def test_documented_give_back_keeps_what_later_tokens_see(spans, block):
    """The recipe of the documents, run as it stands after every step of a row: its prompt in chunks, then tokens one at a
    time, each in the sequence before it is in the pool; layers of several widths share the table."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    texts = [open(path).read() for path in sorted(glob.glob(os.path.join(root, "*.md")))]
    recipes = [x for t in texts for x in re.findall(r"```python\n(.*?)```", t, re.S) if "window_blocks(" in x]
    assert len(recipes) == 1
    recipe = compile(textwrap.dedent(recipes[0]), "recipe", "exec")
    layers = [slo_attn.Attention(8, 128, 0.1, 2, window=w, sinks=s) for w, s in spans]
    # what a recipe that takes one width and one count of sinks is to be given
    names = dict(W=max(w for w, _ in spans), S=max(s for _, s in spans))
    prompt, generated = 700, 200
    seq = Sequence(num_tokens=prompt, num_cached_tokens=0, num_scheduled_tokens=0, block_table=list(range(-(-(prompt + generated) // block))))
    freed = []

    def step(first, count, is_prefill):
        for t in range(first, first + count):
            assert seq.block_table[t // block] >= 0, f"the page that token {t} is written to is gone"
            for w, s in spans:
                seen = owin.visible(1, t + 1, t, w, s)[0].nonzero()[:, 0] // block
                gone = [b for b in seen.unique().tolist() if seq.block_table[b] < 0]
                assert not gone, f"token {t} sees keys of pages {gone}"
        exec(recipe, dict(names, window_blocks=window_blocks, seq=seq, layers=layers, is_prefill=is_prefill,
                          self=SimpleNamespace(block_size=block), free_page=freed.append))

    for count in (300, 33, 367):
        seq.num_scheduled_tokens = count
        step(seq.num_cached_tokens, count, True)
        seq.num_cached_tokens += count
    for t in range(prompt, prompt + generated):
        seq.num_tokens = t + 2  # token t, and the one sampled after it, appended before the recipe runs
        step(t, 1, False)
    end = prompt + generated
    assert len(set(freed)) == len(freed) and sorted(freed) == list(window_blocks(end, names["W"], names["S"], block))


def test_scaled_tables():
    dim, base, trained, n = 64, 1e4, 2048, 9000
    pos = np.arange(n)[:, None].astype(np.float64)
    freq = base ** (-np.arange(0, dim, 2) / dim)

    def same(table, angle, size=1.0):
        want = np.concatenate((np.cos(angle), np.sin(angle)), -1) * size
        # an angle of up to n turns is off by its rounding in 64 bits, the table by one to 32
        assert table.dtype == torch.float32 and np.abs(table.numpy() - want).max() <= 2.0 ** -24 * size + n * 2.0 ** -50

    same(slo_attn.rope_cos_sin(128, n, base, "cpu", rotary_dim=dim), pos * freq)
    same(slo_attn.rope_cos_sin(dim, n, base, "cpu", scaling=dict(rope_type="linear", factor=3.0)), pos * freq / 3)
    table = slo_attn.rope_cos_sin(dim, n, base, "cpu", scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=trained))
    turns = trained * freq / (2 * math.pi)
    at = lambda t: dim * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = math.floor(at(32)), math.ceil(at(1))
    ramp = np.clip((np.arange(dim // 2) - low) / (high - low), 0, 1)
    same(table, pos * freq * (1 - ramp + ramp / 4), 0.1 * math.log(4) + 1)
    size = table[0, 0].item()
    angle = torch.atan2(table[1, dim // 2:], table[1, :dim // 2]).double().numpy()
    assert np.allclose(angle[turns > 36], freq[turns > 36], rtol=1e-6) and (turns > 36).any()
    assert np.allclose(angle[turns < 0.7], freq[turns < 0.7] / 4, rtol=1e-6) and (turns < 0.7).any()
    assert ((angle <= freq * (1 + 1e-6)) & (angle >= freq / 4 * (1 - 1e-6))).all() and abs(size - 1.1386294) < 1e-6
    flat = slo_attn.rope_cos_sin(dim, 10, base, "cpu", scaling=dict(type="yarn", factor=4.0, original_max_position_embeddings=trained,
                                                                     attention_factor=1.0))
    assert flat[0, 0] == 1.0
    # the reference's own table is as it was
    t = torch.arange(50, dtype=torch.float)
    f = torch.einsum("i,j -> ij", t, 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float) / dim)))
    assert torch.equal(slo_attn.rope_cos_sin(dim, 50, base, "cpu"), torch.cat((f.cos(), f.sin()), -1))
    for bad in (dict(rope_type="other", factor=2.0), dict(rope_type="linear", factor=0.5), dict(rope_type="linear", factor=float("nan"))):
        with pytest.raises(ValueError):
            slo_attn.rope_cos_sin(dim, 10, base, "cpu", scaling=bad)
    for dim_ in (0, 130, 63):
        with pytest.raises(ValueError):
            slo_attn.rope_cos_sin(128, 10, base, "cpu", rotary_dim=dim_)


def test_scalings_that_the_table_would_not_follow():
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048)
    slo_attn.rope_cos_sin(64, 10, 1e4, "cpu", scaling=yarn)
    for bad in ({**yarn, "mscale": 0.7}, {**yarn, "truncate": False}, dict(rope_type="yarn", factor=4.0), dict(rope_type="linear"),
                dict(rope_type="linear", factor=2.0, beta_fast=8)):
        with pytest.raises(ValueError, match="takes only"):
            slo_attn.rope_cos_sin(64, 10, 1e4, "cpu", scaling=bad)


def test_scalings_are_followed_or_refused():
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048)
    table = lambda scaling, base=1e4: slo_attn.rope_cos_sin(64, 10, base, "cpu", scaling=scaling)  # noqa: E731
    for bad in (dict(factor=4.0), dict(rope_type="default", factor=4.0), {**yarn, "rope_type": "default"},
                dict(original_max_position_embeddings=2048), {**yarn, "type": "linear"}, dict(rope_type=None, factor=4.0),
                {**yarn, "factor": None}, {**yarn, "factor": "four"}, {**yarn, "factor": 0.0}, {**yarn, "factor": float("inf")},
                {**yarn, "attention_factor": 0.0}, {**yarn, "attention_factor": -1.0}, {**yarn, "attention_factor": float("nan")},
                {**yarn, "original_max_position_embeddings": None}, {**yarn, "original_max_position_embeddings": 0},
                {**yarn, "original_max_position_embeddings": float("inf")}, {**yarn, "beta_fast": 1.0}, {**yarn, "beta_slow": 32},
                {**yarn, "beta_fast": 2, "beta_slow": 8}, {**yarn, "beta_fast": 0}, {**yarn, "beta_slow": -1.0}):
        with pytest.raises(ValueError, match="rope scaling"):
            table(bad)
    with pytest.raises(ValueError, match="base"):
        table(yarn, 1.0)
    # nothing asked for, and what stands for the defaults
    plain = slo_attn.rope_cos_sin(64, 10, 1e4, "cpu", rotary_dim=64)
    for none in ({}, dict(rope_type="default"), dict(type="default", rope_type="default")):
        assert torch.equal(table(none), plain)
    assert torch.equal(table({**yarn, "type": "yarn", "attention_factor": None, "beta_fast": None, "beta_slow": 1}), table(yarn))
    assert not torch.equal(table(yarn), plain)


def attention_args(**over):
    a = _lib.PagedAttentionArgs()
    a.head_dim, a.num_heads, a.num_kv_heads, a.softmax_scale, a.kv_dtype = 128, 32, 8, 0.1, _lib.KV_FP8_E4M3FN
    a.q = a.out = a.k_cache = a.v_cache = a.k_scale = a.v_scale = 4096
    a.q_row_stride = a.out_row_stride = 32 * 128
    a.num_q_rows = a.num_decode = 4
    a.num_blocks, a.block_size, a.phases = 2, 256, 3
    a.decode_lens, a.decode_tables, a.decode_table_stride, a.decode_table_width = 4096, 4096, 16, 16
    for name, value in over.items():
        setattr(a, name, value)
    return a


COLD = dict(num_decode=0, num_prefill=1, prefill_cu_q=4096, prefill_cu_k=4096, k=4096, v=4096, k_row_stride=1024,
            v_row_stride=1024, num_kv_rows=4)


@pytest.mark.parametrize("over,code,word", [
    (dict(head_dim=64), 4, "head_dim"), (dict(num_heads=30), 1, "multiple"), (dict(num_heads=136), 4, "16 query heads"),
    (dict(num_decode=5), 1, "row counts"), (dict(num_decode=-1), 1, "row counts"), (dict(softmax_scale=0.0), 1, "softmax_scale"),
    (dict(softmax_scale=float("inf")), 1, "softmax_scale"), (dict(q=0), 1, "null"), (dict(q=4104), 1, "aligned"),
    (dict(q_row_stride=4100), 1, "aligned"), (dict(k_cache=0), 1, "pool"), (dict(k_scale=0), 1, "scale"),
    (dict(v_scale=4100), 1, "aligned"), (dict(kv_dtype=3), 1, "kv_dtype"), (dict(block_size=96), 4, "block_size"),
    (dict(decode_lens=0), 1, "metadata"), (dict(decode_table_width=0), 1, "metadata"), (dict(num_prefill=1), 1, "metadata"),
    (dict(decode_table_width=1 << 23), 4, "tokens"), (dict(num_decode=40000, num_q_rows=40000), 4, "rows"),
    (dict(num_prefill=1025), 4, "rows"), (dict(store_slot_mapping=4096), 1, "store"),
    (dict(num_heads=4096, num_kv_heads=4096, q_row_stride=1 << 19, out_row_stride=1 << 19, num_decode=8192, num_q_rows=8192), 4, "too many"),
    (dict(COLD, k=0), 1, "need k and v"), (dict(COLD, num_kv_rows=0), 1, "need k and v"), (dict(COLD, v_row_stride=1016), 1, "apart"),
    (dict(COLD, k=4104), 1, "aligned"), (dict(COLD, num_kv_rows=(1 << 24) + 1), 4, "rows"),
    (dict(COLD, prefill_tables=4096), 1, "metadata"),
])
def test_window_refusals_without_a_gpu(over, code, word):
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    for call in (lambda a: lib.slo_paged_attention_window(bytes(a), 100, 4, None),
                 lambda a: lib.slo_paged_attention_window_workspace_bytes(bytes(a), 100, 4, ctypes.byref(need))):
        assert call(attention_args(**over)) == code
        assert word in lib.slo_last_error().decode()


def test_window_sizes_without_a_gpu():
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    size = lambda a, w, s: lib.slo_paged_attention_window_workspace_bytes(bytes(a), w, s, ctypes.byref(need))  # noqa: E731
    for window, sinks in ((0, 4), (-1, 0), (5, -1)):
        assert lib.slo_paged_attention_window(bytes(attention_args()), window, sinks, None) == 1
        assert size(attention_args(), window, sinks) == 1
    assert lib.slo_paged_attention_window(None, 5, 0, None) == 1
    assert lib.slo_paged_attention_window_workspace_bytes(bytes(attention_args()), 5, 0, None) == 1
    # nothing to do
    assert lib.slo_paged_attention_window(bytes(attention_args(num_decode=0)), 5, 0, None) == 0
    # a row with a wide window is cut and needs a workspace, under a narrow one, however wide its table, it does not
    a = attention_args(decode_table_width=4096, num_decode=1)
    assert size(a, 1 << 30, 1 << 30) == 0 and need.value > 0
    assert lib.slo_paged_attention_window(bytes(a), 1 << 30, 0, None) == 3
    a.workspace, a.workspace_bytes = 4096, need.value - 1
    assert lib.slo_paged_attention_window(bytes(a), 1 << 30, 1 << 30, None) == 3
    assert size(a, 64, 0) == 0 and need.value == 0


def test_rope_store_refusals_without_a_gpu():
    lib = _lib.load()

    def call(**over):
        a = _lib.RopeStoreArgs()
        a.num_tokens, a.num_heads, a.num_kv_heads, a.head_dim, a.rotary_dim, a.interleaved = 4, 32, 8, 128, 64, 1
        a.qkv_row_stride, a.eps, a.max_position, a.kv_dtype, a.num_slots, a.scale_floor = 6144, 1e-6, 100, 1, 100, 2.0 ** -64
        for name, kind in a._fields_:
            if kind is ctypes.c_void_p:
                setattr(a, name, 4096)
        for name, value in over.items():
            setattr(a, name, value)
        return lib.slo_rope_store(bytes(a), None)

    assert lib.slo_rope_store(None, None) == 1 and call(num_tokens=0) == 0
    for over in (dict(num_tokens=-1), dict(num_heads=0), dict(num_kv_heads=0), dict(q_norm_weight=None), dict(eps=-1.0),
                 dict(eps=float("nan")), dict(max_position=0), dict(rotary_dim=0), dict(rotary_dim=60), dict(rotary_dim=136),
                 dict(kv_dtype=2), dict(qkv=None), dict(qkv=4104), dict(qkv_row_stride=6136), dict(qkv_row_stride=6148),
                 dict(cos_sin=4100), dict(k_scale=None), dict(scale_floor=0.0), dict(num_slots=-1), dict(k_cache=None),
                 dict(k_cache=4104), dict(slot_mapping=None)):
        assert call(**over) == 1, over
    assert call(head_dim=96) == 4 and call(num_heads=65537, qkv_row_stride=1 << 24) == 4


def test_packed_rope_arguments_are_the_struct():
    a = _lib.RopeStoreArgs()
    for i, (name, _) in enumerate(a._fields_, 1):
        setattr(a, name, i)
    assert _lib.pack_rope_args(*range(1, len(a._fields_) + 1)) == bytes(a)


def test_layer_refuses_a_window_that_is_none():
    for window, sinks in ((-1, 0), (0, 3), (5, -1)):
        with pytest.raises(ValueError):
            slo_attn.Attention(8, 128, 0.1, 2, window, sinks)
    layer = slo_attn.Attention(8, 128, 0.1, 2)
    assert layer.window == 0 and layer.sinks == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        slo_attn.paged_attention(torch.zeros(1, 8, 128, dtype=torch.bfloat16), None, None, 0.1, num_kv_heads=2, window=5, num_prefill=1,
                                 prefill_cu_q=torch.zeros(2, dtype=torch.int32), prefill_cu_k=torch.zeros(2, dtype=torch.int32))
