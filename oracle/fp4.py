"""4-bit KV format -- CPU definition.

Codes are E2M1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2,
3, 4, 6), two to a byte with the even channel in the low half; every 32
channels of a (token, kv head) vector share an E8M0 scale, a power of two
biased by 127.  ``quantize_kv``:

    amax  = max|x| over the 32 channels (infinities and NaN as the largest
            finite bf16)
    scale = the smallest power of two in [scale_floor, 2^125] with
            amax < 7 * scale, or 2^125
    code  = the E2M1 value nearest to x / scale, ties to the even code,
            saturating at 6; the sign is kept, also for zeros

The reference plans no 4-bit cache; element and scale formats are those of the
OCP Microscaling specification, the scale rule is this library's own (the
specification's puts amax / scale in [4, 8), so up to a quarter of the largest
value is lost to saturation).
"""
from __future__ import annotations

import numpy as np

GROUP = 32
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=np.float64)
SCALE_FLOOR = 2.0 ** -64
BF16_MAX = float(np.uint32(0x7F7F0000).view(np.float32))


def quantize_kv(x: np.ndarray, scale_floor: float = SCALE_FLOOR):
    """``x`` [..., D] (bf16 values as float32) -> (bytes uint8 [..., D/2], scales uint8 [..., D/32])."""
    x = np.asarray(x, dtype=np.float32)
    sign = np.signbit(x)
    mag = np.abs(np.where(np.isfinite(x), x, np.float32(BF16_MAX)).astype(np.float64))
    mag = mag.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    amax = mag.max(axis=-1)
    lo, hi = int(np.log2(scale_floor)), 125
    exponent = np.full(amax.shape, lo, dtype=np.int64)
    for e in range(lo, hi):
        exponent = np.where(amax >= 7.0 * 2.0 ** e, e + 1, exponent)
    y = mag * np.exp2(-exponent.astype(np.float64))[..., None]
    d = np.abs(y[..., None] - VALUES)
    near = d == d.min(axis=-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)).reshape(x.shape) + 8 * sign
    return (code[..., 0::2] + 16 * code[..., 1::2]).astype(np.uint8), (exponent + 127).astype(np.uint8)


def dequantize_kv(packed: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 values [..., D] of bytes [..., D/2] and scales [..., D/32]."""
    code = np.stack((packed & 15, packed >> 4), axis=-1).reshape(*packed.shape[:-1], 2 * packed.shape[-1])
    v = np.where(code & 8, -1.0, 1.0) * VALUES[code & 7]
    s = np.exp2(scale.astype(np.float64) - 127.0)
    return (v.reshape(*scale.shape, GROUP) * s[..., None]).reshape(code.shape)


def store_kvcache(key, value, k_pages, v_pages, k_scale, v_scale, slot_mapping, scale_floor: float = SCALE_FLOOR):
    """Writes rows [N, H, D] into pages [blocks, H, block_size, D/2] and scales [blocks, H, block_size, D/32]."""
    block = k_pages.shape[2]
    for src, pages, scales in ((key, k_pages, k_scale), (value, v_pages, v_scale)):
        codes, sc = quantize_kv(src, scale_floor)
        for i, slot in enumerate(slot_mapping):
            if 0 <= slot < pages.shape[0] * block:
                pages[slot // block, :, slot % block] = codes[i]
                scales[slot // block, :, slot % block] = sc[i]
