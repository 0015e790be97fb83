"""Rotary layouts, norms and the KV write in one call on the GPU, against the
formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

import slo_attn
from fp4_cases import i32
from oracle import fp4 as ofp4
from oracle import fp8 as ofp8

pytestmark = pytest.mark.gpu
EPS = 1e-6


def definition(x, w, table, pos, rot, interleaved):
    """fp64 (result, bound) of heads x [n, H, D]; table [max_position, rot]."""
    y = x.double()
    rel = 0.0
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
        # a sum of D squares in fp32, its mean, rsqrt within an ulp, two products
        rel = (x.shape[-1] + 8) * 2.0 ** -24
    t = table[pos.clamp(0, len(table) - 1)].double()[:, None]
    c, s = t[..., :rot // 2], t[..., rot // 2:]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, size = y.clone(), y.abs()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    size[..., a], size[..., b] = (y[..., a] * c).abs() + (y[..., b] * s).abs(), (y[..., b] * c).abs() + (y[..., a] * s).abs()
    # two products and a sum in fp32, then one rounding to bf16
    return out, ((rel + 3 * 2.0 ** -24) * size * (1 + 2.0 ** -8) + 2.0 ** -8 * out.abs()) * 1.01 + 1e-38


def pools(fmt, blocks, block, hkv, d, device):
    if fmt == "fp4":
        shape, sc = (blocks, hkv, block, d // 2), torch.full((blocks, hkv, block, d // 32), 0xFF, dtype=torch.uint8, device=device)
        return [torch.full(shape, 0xA5, dtype=torch.uint8, device=device) for _ in range(2)], [sc, sc.clone()]
    if fmt == "fp8":
        sc = torch.full((blocks, block, hkv), 9.0, device=device)
        return [torch.full((blocks, block, hkv, d), 0x35, dtype=torch.uint8, device=device) for _ in range(2)], [sc, sc.clone()]
    return [torch.full((blocks, block, hkv, d), 5.0, dtype=torch.bfloat16, device=device) for _ in range(2)], [None, None]


def as_pool(t, fmt):
    return t.view(torch.float4_e2m1fn_x2) if fmt == "fp4" else t


def check_pool(fmt, side, scale, tokens, slots, block):
    """The pool holds ``tokens`` at their slots, quantised as the stores quantise, and what it held elsewhere."""
    got, sc = side.cpu(), None if scale is None else scale.cpu()
    want_p, want_s = pools(fmt, len(got), block, tokens.shape[1], tokens.shape[2], "cpu")
    want, ws = want_p[0], want_s[0]
    for i, slot in enumerate(slots):
        if not 0 <= slot < len(got) * block:
            continue
        x = tokens[i].float().cpu()
        if fmt == "bf16":
            want[slot // block, slot % block] = tokens[i].cpu()
        elif fmt == "fp8":
            codes, s = ofp8.quantize_kv(x.numpy()[None])
            want[slot // block, slot % block], ws[slot // block, slot % block] = torch.from_numpy(codes[0]), torch.from_numpy(s[0])
        else:
            codes, s = ofp4.quantize_kv(x.numpy()[None])
            want[slot // block, :, slot % block], ws[slot // block, :, slot % block] = torch.from_numpy(codes[0]), torch.from_numpy(s[0])
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    assert sc is None or torch.equal(sc.view(torch.uint8), ws.view(torch.uint8))


CASES = [  # tokens, hq, hkv, d, rot, interleaved, norm
    (1, 1, 1, 64, 8, True, True), (1, 32, 8, 128, 64, False, True), (37, 32, 8, 128, 128, True, True),
    (37, 5, 1, 128, 128, False, False), (9, 7, 3, 128, 96, False, True), (9, 7, 3, 128, 8, False, True),
    (13, 8, 8, 256, 256, False, True), (13, 8, 2, 256, 200, True, False), (20, 40, 12, 64, 64, False, True),
    (20, 3, 2, 64, 40, True, True), (5, 64, 8, 128, 72, False, True), (300, 28, 4, 128, 120, True, True),
]


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("n,hq,hkv,d,rot,interleaved,norm", CASES)
def test_layouts(device, fmt, n, hq, hkv, d, rot, interleaved, norm):
    g = torch.Generator().manual_seed(n + rot)
    block, far = 64, 1000
    wide = (torch.randn(n, hq + 2 * hkv + 1, d, generator=g) * 3).to(torch.bfloat16).flatten(1).to(device)
    qkv = wide[:, :-d]  # rows of a wider buffer
    pos = torch.randint(0, far, (n,), generator=g)
    blocks = -(-n // block) + 1
    slots = torch.randperm(blocks * block, generator=g)[:n].tolist()
    if n >= 9:
        pos[1], pos[2], pos[3] = far + 5, -3, far - 1  # clamped into the table
        slots[4], slots[5] = -1, blocks * block        # not in the pool
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(torch.bfloat16).to(device) if norm else None for _ in range(2)]
    table = slo_attn.rope_cos_sin(d, far, 1e4, device, rotary_dim=rot)
    side, scale = pools(fmt, blocks, block, hkv, d, device)
    q, k, v = slo_attn.qk_norm_rope_store(qkv, pos.to(device), w[0], w[1], EPS, table, hq, hkv, as_pool(side[0], fmt),
                                          as_pool(side[1], fmt), i32(slots, device), *scale, head_dim=d, rotary_dim=rot,
                                          interleaved=interleaved)
    x = qkv.view(n, hq + 2 * hkv, d).cpu()
    for got, heads, weight in ((q, x[:, :hq], w[0]), (k, x[:, hq:hq + hkv], w[1])):
        want, bound = definition(heads, None if weight is None else weight.cpu(), table.cpu(), pos, rot, interleaved)
        off = (got.double().cpu() - want).abs()
        assert (off <= bound).all(), f"{(off / bound).max():.3f} of the bound"
    assert torch.equal(v.cpu(), x[:, hq + hkv:]) and v.data_ptr() == qkv[:, (hq + hkv) * d:].data_ptr()
    check_pool(fmt, side[0], scale[0], k, slots, block)
    check_pool(fmt, side[1], scale[1], v, slots, block)


def test_more_tokens_than_a_grid_and_none(device):
    n, d = (1 << 20) + 3, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(n, 3 * d, generator=g, device=device).to(torch.bfloat16)
    pos = torch.arange(n, device=device) % 100
    table = slo_attn.rope_cos_sin(d, 100, 1e4, device, rotary_dim=d)
    side, _ = pools("bf16", -(-n // 64), 64, 1, d, device)
    slots = torch.arange(n, dtype=torch.int32, device=device)
    run = lambda a, b: slo_attn.qk_norm_rope_store(qkv[a:b], pos[a:b], None, None, 0.0, table, 1, 1, side[0], side[1],  # noqa: E731
                                                   slots[a:b], head_dim=d)
    q, k, _ = run(0, n)
    pool = side[0].flatten(0, 1)[:n].clone()
    assert torch.equal(pool, k)
    for a in (0, 500_000, n - 5):
        q2, k2, _ = run(a, min(a + 300, n))
        assert torch.equal(q2, q[a:a + 300]) and torch.equal(k2, k[a:a + 300])
    assert run(5, 5)[0].shape == (0, 1, d)


def test_values_over_the_exponent_range(device):
    # rows whose squares vanish beside eps, are zero, or sum past fp32 (as rsqrt(inf): zeros), and NaN stays in its own head
    d, hq, hkv = 128, 2, 1
    g = torch.Generator().manual_seed(3)
    x = torch.randn(8, 4, d, generator=g)
    x[0] *= 2.0 ** -60
    x[1] = 0
    x[2] *= 2.0 ** 50
    x[3] *= 2.0 ** 100
    x[4, 0, 7] = float("nan")
    x[5, 1, 3] = float("inf")
    x = x.to(torch.bfloat16)
    w = torch.ones(d, dtype=torch.bfloat16, device=device)
    table = slo_attn.rope_cos_sin(d, 16, 1e4, device, rotary_dim=d)
    side, _ = pools("bf16", 1, 64, hkv, d, device)
    pos = torch.arange(8, device=device)
    q, k, _ = slo_attn.qk_norm_rope_store(x.flatten(1).to(device), pos, w, w, EPS, table, hq, hkv, side[0], side[1],
                                          i32(range(8), device), interleaved=True)
    want, bound = definition(x[:, :2], w.cpu(), table.cpu(), pos.cpu(), d, True)
    fine = torch.ones(8, 2, dtype=torch.bool)
    fine[3], fine[4, 0], fine[5, 1] = False, False, False
    assert ((q.double().cpu() - want).abs() <= bound)[fine].all()
    assert not q[3].any() and q[4, 0].isnan().all() and torch.isfinite(q[5, 0]).all()


def test_scaled_tables_and_the_reference_layout(device):
    # a table scaled for long contexts serves the reference's layout too, with that path's roundings
    d, n, hq, hkv = 128, 50, 8, 2
    scaling = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=512)
    table = slo_attn.rope_cos_sin(d, 2048, 1e4, device, scaling=scaling)
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 2048, (n,), generator=g)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16)
    side, _ = pools("bf16", 1, 64, hkv, d, device)
    q, _, _ = slo_attn.qk_norm_rope_store(qkv.to(device), pos.to(device), w.to(device), w.to(device), EPS, table, hq, hkv,
                                          side[0], side[1], i32(range(n), device))
    x = qkv.view(n, -1, d)[:, :hq]
    want, bound = definition(x, w, table.cpu(), pos, d, False)
    size = want.abs() + torch.cat((want[..., d // 2:], want[..., :d // 2]), -1).abs()
    # two more roundings to bf16, of the normed head and of its product with the weight, each of up to 2^-8 of a pair's values
    assert ((q.double().cpu() - want).abs() <= bound + 2 * 2.0 ** -8 * 1.02 * math.sqrt(2) * size + 2.0 ** -14 * size).all()


def test_refusals(device):
    d, hq, hkv = 128, 4, 2
    qkv = torch.zeros(3, 8 * d, dtype=torch.bfloat16, device=device)
    pos = torch.zeros(3, dtype=torch.int64, device=device)
    w = torch.ones(d, dtype=torch.bfloat16, device=device)
    table = slo_attn.rope_cos_sin(d, 16, 1e4, device, rotary_dim=64)
    side, _ = pools("bf16", 1, 64, hkv, d, device)
    slots = i32([0, 1, 2], device)

    def call(qkv=qkv, pos=pos, qw=w, kw=w, table=table, hq=hq, kc=side[0], vc=side[1], slots=slots, ks=None, vs=None, **over):
        return slo_attn.qk_norm_rope_store(qkv, pos, qw, kw, EPS, table, hq, hkv, kc, vc, slots, ks, vs, **{"rotary_dim": 64, **over})

    call()
    for error, over in ((ValueError, dict(rotary_dim=60)), (ValueError, dict(rotary_dim=0)), (ValueError, dict(rotary_dim=136)),
                        (ValueError, dict(rotary_dim=128, interleaved=True)), (ValueError, dict(qw=None)), (ValueError, dict(kw=w[:64])),
                        (ValueError, dict(kw=w.float())), (ValueError, dict(hq=5)), (TypeError, dict(qkv=qkv.float())),
                        (ValueError, dict(pos=pos.int())), (ValueError, dict(pos=pos[:2])), (ValueError, dict(slots=slots[:2])),
                        (ValueError, dict(slots=slots.long())), (ValueError, dict(table=table.double())),
                        (ValueError, dict(kc=side[0][:, :, :1])), (ValueError, dict(vc=side[1].view(1, 32, 4, d))),
                        (TypeError, dict(kc=side[0].view(torch.uint8))), (RuntimeError, dict(slots=slots.cpu())),
                        (ValueError, dict(head_dim=64))):
        with pytest.raises(error):
            call(**over)
    with pytest.raises(RuntimeError, match="head_dim"):
        wide = torch.zeros(1, 64, 2, 32, dtype=torch.bfloat16, device=device)
        call(qkv=qkv[:, :256], kc=wide, vc=wide.clone(), head_dim=32, rotary_dim=32, qw=None, kw=None,
             table=slo_attn.rope_cos_sin(32, 16, 1e4, device, rotary_dim=32))
    assert np.isfinite(side[0].float().cpu().numpy()).all()
