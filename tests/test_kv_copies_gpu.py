"""Many tokens at once into a 4-bit pool, and read back from any: 16,384 tokens
and more, where a workgroup takes four of them if their heads are few, and read
backs of more than the last-level cache holds."""
import numpy as np
import pytest
import torch

import slo_attn
from fp4_cases import STALE, i32, random_values
from oracle import fp4 as ofp4
from oracle import fp8 as ofp8

pytestmark = pytest.mark.gpu

# (tokens, kv heads, head_dim): every remainder of four, one token over less than, just and more than a workgroup's lanes
MANY = [(16384, 1, 64), (16385, 3, 128), (16386, 8, 128), (16387, 2, 256), (16387, 8, 64), (16385, 9, 128), (16386, 8, 256),
        (16383, 2, 128)]
BASE = 257  # different tokens; the rest repeat them


def scattered(n, block, g):
    """A pool's block count, and different slots for n tokens, a few of them outside it."""
    blocks = n // block + 3
    slots = torch.randperm(blocks * block, generator=g)[:n].int()
    slots[[0, 5, n // 2, n - 1]] = torch.tensor([-1, blocks * block, -9, blocks * block + 7], dtype=torch.int32)
    return blocks, slots


@pytest.mark.parametrize("n,hkv,d", MANY)
def test_store_of_many_tokens(device, n, hkv, d):
    g = torch.Generator().manual_seed(n + hkv)
    block = 192
    blocks, slots = scattered(n, block, g)
    qkv = random_values(g, BASE, 2 * hkv + 1, d)
    token = torch.arange(n) % BASE
    dev = qkv.to(device)[token.to(device)]
    pages = [torch.full((blocks, hkv, block, d // 2), 0xA5, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.full((blocks, hkv, block, d // 32), STALE, dtype=torch.uint8, device=device) for _ in range(2)]
    slo_attn.store_kvcache(dev[:, 1:1 + hkv], dev[:, 1 + hkv:], *(p.view(torch.float4_e2m1fn_x2) for p in pages),
                           slots.to(device), *scales)
    live = (slots >= 0) & (slots < blocks * block)
    page, off = slots[live].long() // block, slots[live].long() % block
    for side, x in enumerate((qkv[:, 1:1 + hkv], qkv[:, 1 + hkv:])):
        codes, scale = (torch.from_numpy(t) for t in ofp4.quantize_kv(x.float().numpy()))
        want_p, want_s = torch.full(pages[side].shape, 0xA5, dtype=torch.uint8), torch.full(scales[side].shape, STALE, dtype=torch.uint8)
        want_p[page, :, off] = codes[token[live]]
        want_s[page, :, off] = scale[token[live]]
        assert torch.equal(pages[side].cpu(), want_p) and torch.equal(scales[side].cpu(), want_s)


def filled(fmt, blocks, block, hkv, d, g, device):
    """A pool of random bytes: (pages, scales) of K and V, and the bf16 values that its tokens stand for, in a table by slot."""
    out = []
    for _ in range(2):
        if fmt == "bf16":
            pages = torch.randn(blocks, block, hkv, d, generator=g, device=device).to(torch.bfloat16)
            scale, value = None, pages.flatten(0, 1)
        elif fmt == "fp8":
            pages = torch.randint(0, 255, (blocks, block, hkv, d), generator=g, dtype=torch.uint8, device=device)
            pages[pages == 0x7F] = 0x7E  # no NaN
            scale = torch.rand(blocks, block, hkv, generator=g, device=device) + 0.01
            code = torch.from_numpy(ofp8.decode_array(np.arange(256, dtype=np.uint8)).astype(np.float32)).to(device)
            value = (code[pages.int()] * scale[..., None]).to(torch.bfloat16).flatten(0, 1)
        else:
            pages = torch.randint(0, 256, (blocks, hkv, block, d // 2), generator=g, dtype=torch.uint8, device=device)
            scale = torch.randint(100, 150, (blocks, hkv, block, d // 32), generator=g, dtype=torch.uint8, device=device)
            code = torch.from_numpy(np.concatenate((ofp4.VALUES, -ofp4.VALUES)).astype(np.float32)).to(device)
            x = torch.stack((code[(pages & 15).int()], code[(pages >> 4).int()]), -1).flatten(-2)
            x = x * torch.exp2(scale.float() - 127).repeat_interleave(32, -1)
            value = x.to(torch.bfloat16).transpose(1, 2).flatten(0, 1)
        out.append((pages.view(torch.float4_e2m1fn_x2) if fmt == "fp4" else pages, scale, value))
    return out


# past the cache: 2 n hkv d 2 bytes from 2^28 on, for the quantised pools
LOADS = MANY + [(65537, 8, 128), (32771, 8, 256), (131073, 4, 128), (65538, 9, 128)]


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("n,hkv,d", LOADS)
def test_read_back_of_many_tokens(device, fmt, n, hkv, d):
    g = torch.Generator(device=device).manual_seed(n + d)
    block, blocks = 64, 19
    (kc, ks, kv), (vc, vs, vv) = filled(fmt, blocks, block, hkv, d, g, device)
    slots = torch.randint(0, blocks * block, (n,), generator=g, device=device).int()
    slots[[0, 6, n // 3, n - 1]] = i32([-1, blocks * block, -5, blocks * block + 1], device)
    live = (slots >= 0) & (slots < blocks * block)
    for got, value in zip(slo_attn.load_kvcache(kc, vc, slots, ks, vs), (kv, vv)):
        want = value[slots.long().clamp(0, blocks * block - 1)]
        want[~live] = 0
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_read_back_of_more_tokens_than_a_grid_of_single_ones_holds(device):
    # 2^24 workgroups of 256 threads are more than a grid may have; 9 heads of 64 channels would take one a token
    n, block, blocks, hkv, d = (1 << 24) + 3, 64, 19, 9, 64
    g = torch.Generator(device=device).manual_seed(4)
    (kc, _, kv), (vc, _, vv) = filled("bf16", blocks, block, hkv, d, g, device)
    slots = torch.randint(0, blocks * block, (n,), generator=g, device=device).int()
    for got, value in zip(slo_attn.load_kvcache(kc, vc, slots), (kv, vv)):
        for part in (slice(0, 5000), slice(n // 2, n // 2 + 5000), slice(n - 5000, n)):
            assert torch.equal(got[part], value[slots[part].long()])
    del got
    torch.cuda.empty_cache()
