"""Limits of the 4-bit attention and of the accumulated weights, on the CPU: what
the C entries size and refuse."""
import ctypes

import pytest
import torch

from slo_attn import _lib
from slo_attn.attention import _pages_of_slots
from test_kv_compress_host import attention_args


def prefill_args(queries, rows, width, heads=32, kv_heads=8, **over):
    return attention_args(**{**dict(num_decode=0, num_q_rows=queries, num_prefill=rows, prefill_cu_q=4096, prefill_cu_k=4096,
                                    prefill_tables=4096, prefill_table_stride=width, prefill_table_width=width,
                                    num_heads=heads, num_kv_heads=kv_heads, q_row_stride=heads * 128,
                                    out_row_stride=heads * 128), **over})


def workspace(call, a):
    need = ctypes.c_size_t(0)
    assert call(bytes(a), ctypes.byref(need)) == 0, _lib.load().slo_last_error()
    return need.value


@pytest.mark.parametrize("bounds", [(0, 0), (0, 900), (700, 0), (1, 1)])
def test_4_bit_prefill_rows_have_a_plan_whatever_the_bounds(bounds):
    call = _lib.load().slo_paged_attention_fp4_workspace_bytes
    exact = workspace(call, prefill_args(700, 2, 16, max_q=700, max_k=900))
    assert exact > 0 and workspace(call, prefill_args(700, 2, 16, max_q=bounds[0], max_k=bounds[1])) > 0


@pytest.mark.parametrize("bounds", [(0, 0), (0, 900), (700, 0), (1, 1), (1 << 17, 1 << 21)])
def test_weights_keep_a_place_for_every_query_whatever_the_bounds(bounds):
    call = _lib.load().slo_accumulate_attention_workspace_bytes
    exact = workspace(call, prefill_args(700, 2, 16, max_q=700, max_k=900))
    assert exact >= 700 * 32 * 4 and workspace(call, prefill_args(700, 2, 16, max_q=bounds[0], max_k=bounds[1])) == exact


@pytest.mark.parametrize("heads,kv_heads,rows,most", [(64, 4, 1, 131071), (64, 4, 129, 130047), (32, 8, 1, 524287), (28, 4, 7, 262047)])
def test_4_bit_prefill_steps_stay_in_32_bits(heads, kv_heads, rows, most):
    # Tiles of 4 floor(32 / group) queries, and one more a row, times 65,536 steps of 64 keys: 2^30 at most, so 2^14 tiles.
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    for n in (most, most + 1):
        a = prefill_args(n, rows, 16384, heads, kv_heads)
        rc = lib.slo_paged_attention_fp4_workspace_bytes(bytes(a), ctypes.byref(need))
        assert rc == (0 if n == most else 4), lib.slo_last_error()
        if rc:
            assert lib.slo_paged_attention_fp4(bytes(a), None) == 4 and b"2^30" in lib.slo_last_error()
    # a captured step's capacities are far below
    assert lib.slo_paged_attention_fp4_workspace_bytes(bytes(prefill_args(65536, 1024, 640)), ctypes.byref(need)) == 0


@pytest.mark.parametrize("lens,block", [([1], 64), ([130, 0, 64, 65], 64), ([300, 17], 128), ([0, 0], 64)])
def test_pages_of_a_cold_prompts_slots(lens, block):
    pages = [-(-n // block) for n in lens]
    order, tables = list(range(40))[::-1], []
    width = max(pages + [1])
    for n in pages:
        tables.append([order.pop(0) for _ in range(n)] + [-1] * (width - n))
    slots = torch.tensor([t[j // block] * block + j % block for t, n in zip(tables, lens) for j in range(n)], dtype=torch.int32)
    cu_k = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)
    got = _pages_of_slots(slots, cu_k, max(lens), block)
    assert got.dtype == torch.int32 and got.tolist() == tables
    # tokens that were not stored are in no page; padding behind the last row is no row's
    if slots.numel():
        padded = torch.cat((torch.full_like(slots, -1), slots))
        assert (_pages_of_slots(padded[:slots.numel()], cu_k, max(lens), block) == -1).all()
        assert _pages_of_slots(torch.cat((slots, slots)), cu_k, max(lens), block).tolist() == tables
        unbounded = _pages_of_slots(slots, cu_k, 0, block)
        assert unbounded[:, :width].tolist() == tables and (unbounded[:, width:] == -1).all()


@pytest.mark.parametrize("kv_dtype,row_bytes", [(0, 256), (1, 128), (2, 64)])
def test_few_long_decode_rows_are_cut(kv_dtype, row_bytes):
    # one launch and no workspace below 512 KiB of K a (row, kv head), or where these fill the CUs
    call = _lib.load().slo_accumulate_attention_workspace_bytes

    def need(rows, tokens):
        return workspace(call, attention_args(num_decode=rows, num_q_rows=rows, decode_table_width=tokens // 64, block_size=64,
                                              num_heads=8, q_row_stride=8 * 128, kv_dtype=kv_dtype))

    long = (512 << 10) // row_bytes
    assert need(1, long - 64) == 0 and need(31, long - 64) == 0 and need(32, long) == 0 and need(32, 16384) == 0
    for rows in (1, 31):
        assert need(rows, long) >= rows * 8 * long * 4
    assert need(32, 16384 + 64) > 0
