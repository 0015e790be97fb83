"""Limits of the compressed KV cache's operators on the GPU: bounds left out or
too small, and what lies past 32 bits."""
import pytest
import torch

import slo_attn
from fp4_cases import Rows
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
