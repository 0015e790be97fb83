"""Limits of the compressed KV cache's operators on the GPU: bounds left out or
too small, and what lies past 32 bits."""
import pytest
import torch

import slo_attn
from fp4_cases import Rows
from test_fp4_gpu import CASES

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
