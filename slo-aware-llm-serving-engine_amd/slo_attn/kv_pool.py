"""KV pool allocation for bf16, E4M3FN or 4-bit caches, and the block lifecycle helpers.

The runner's allocate_kv_cache (nanovllm/engine/model_runner.py:103-121,
nanovllm/engine/mixed_model_runner.py:17-47) sizes the pool by

    block_bytes = 2 * layers * block_size * kv_heads * head_dim * itemsize
    blocks = (total * gpu_memory_utilization - used - peak + current) // block_bytes

and hands each attention layer the views ``pool[0, l]`` / ``pool[1, l]`` of
one ``[2, layers, blocks, block_size, kv_heads, head_dim]`` tensor.  The
quantised pool of docs/project_manual.md:527-563,583 keeps that layout with
E4M3FN code bytes and adds one fp32 scale per (token, kv head), K and V each:
``[2, layers, blocks, block_size, kv_heads]`` (the scale layout of
docs/project_manual.md:174-189), so a block costs
``2 * layers * block_size * kv_heads * (head_dim + 4)`` bytes instead of
``... * head_dim * 2`` -- 264 against 512 bytes per token and kv head at
head_dim 128 (docs/project_manual.md:548-556).

The 4-bit pool (E2M1 codes, two to a byte, with one E8M0 scale byte per 32
channels) stores its pages head by head, ``[2, layers, blocks, kv_heads,
block_size, head_dim / 2]`` and ``[..., head_dim / 32]``: 136 bytes per token
and kv head at head_dim 128.  With ``track_scores`` a pool also keeps every
cached token's accumulated attention weight per kv head, fp32 ``[layers,
blocks, kv_heads, block_size]``, which ``Attention`` adds to and ``evict``
reads.

Lifecycle (docs/project_manual.md:591-602): a block's code bytes and scales
are one cache object, so copying a block (copy-on-write of a shared tail) or
snapshotting it moves both, and a block taken back into use has its scales
reset with its bytes; accumulated weights move and are reset with them.  The store kernels write every (token, kv head) scale
together with its codes, and attention reads only tokens below a row's
length, so stale scales beyond a row's valid tokens are never read.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import evict_kv, load_kvcache

_KV_FORMATS = {"bf16": _lib.KV_BF16, "fp8_e4m3fn": _lib.KV_FP8_E4M3FN, "fp4_e2m1": _lib.KV_FP4_E2M1}


def kv_block_bytes(num_layers: int, block_size: int, num_kv_heads: int, head_dim: int,
                   kv_format: str = "bf16", track_scores: bool = False) -> int:
    """Bytes of one block across all layers, K and V, scales (and accumulated weights) included."""
    vectors = num_layers * block_size * num_kv_heads
    scores = 4 * vectors if track_scores else 0
    if kv_format == "bf16":
        return 2 * vectors * head_dim * 2 + scores
    if kv_format == "fp8_e4m3fn":
        return 2 * vectors * (head_dim + 4) + scores
    if kv_format == "fp4_e2m1":
        return 2 * vectors * (head_dim // 2 + head_dim // _lib.FP4_GROUP) + scores
    raise ValueError(f"unknown KV format {kv_format!r}")


def num_kv_blocks(total: int, used: int, peak: int, current: int, gpu_memory_utilization: float,
                  block_bytes: int, cap: int | None = None) -> int:
    """Block count of allocate_kv_cache (mixed_model_runner.py:20-33), optionally capped."""
    count = int(total * gpu_memory_utilization - used - peak + current) // block_bytes
    if cap is not None:
        count = min(count, cap)
    return count


def window_blocks(length: int, window: int, sinks: int, block_size: int) -> range:
    """Places in the block table of a row of ``length`` cached tokens whose pages no later token sees.

    A token at position t >= ``length`` sees the keys j > t - window and j <
    sinks.  An engine gives these pages back (or to another row) and puts -1 in
    their places: attention with the window does not read them.  ``length``
    counts the tokens whose K and V are in the pool: neither a sampled token
    that is not yet there nor the rest of a prompt that comes in chunks; with
    either, pages that the next tokens see would go, and nothing would say so.
    Where layers share the table, ``window`` and ``sinks`` are the largest of
    theirs."""
    if window <= 0 or sinks < 0 or block_size <= 0:
        raise ValueError("window and block_size must be positive and sinks not negative")
    return range(-(-sinks // block_size), max(length - window + 1, 0) // block_size)


class KVPool:
    """One pool for all layers: codes or bf16 values, and the scales of the quantised formats.

    ``kv``    ``[2, layers, blocks, block_size, kv_heads, head_dim]`` bf16 or uint8;
              4 bits: ``[2, layers, blocks, kv_heads, block_size, head_dim / 2]`` uint8
    ``scale`` ``[2, layers, blocks, block_size, kv_heads]`` fp32 (E4M3FN);
              ``[2, layers, blocks, kv_heads, block_size, head_dim / 32]`` uint8 (4 bits)
    ``scores`` ``[layers, blocks, kv_heads, block_size]`` fp32 (``track_scores``)
    """

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 kv_format: str = "bf16", device=None, track_scores: bool = False):
        if kv_format not in _KV_FORMATS:
            raise ValueError(f"unknown KV format {kv_format!r}")
        if num_blocks <= 0:
            raise RuntimeError("no KV blocks available")
        self.kv_format = kv_format
        self.num_layers, self.num_blocks, self.block_size = num_layers, num_blocks, block_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        shape = (2, num_layers, num_blocks, block_size, num_kv_heads, head_dim)
        if kv_format == "bf16":
            self.kv = torch.empty(shape, dtype=torch.bfloat16, device=device)
            self.scale = None
        elif kv_format == "fp8_e4m3fn":
            self.kv = torch.zeros(shape, dtype=torch.uint8, device=device)
            self.scale = torch.ones(shape[:-1], dtype=torch.float32, device=device)
        else:
            if head_dim % _lib.FP4_GROUP:
                raise ValueError(f"a 4-bit pool needs a head_dim that is a multiple of {_lib.FP4_GROUP}")
            shape = (2, num_layers, num_blocks, num_kv_heads, block_size)
            self.kv = torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device)
            self.scale = torch.full((*shape, head_dim // _lib.FP4_GROUP), 127, dtype=torch.uint8, device=device)
        self.scores = None
        if track_scores:
            self.scores = torch.zeros((num_layers, num_blocks, num_kv_heads, block_size), dtype=torch.float32, device=device)

    @classmethod
    def for_memory(cls, num_layers: int, block_size: int, num_kv_heads: int, head_dim: int, kv_format: str,
                   gpu_memory_utilization: float = 0.9, cap: int | None = None, device=None,
                   track_scores: bool = False) -> "KVPool":
        """Sizes the pool from the device's free memory like allocate_kv_cache."""
        device = torch.device(device if device is not None else "cuda")
        free, total = torch.cuda.mem_get_info(device)
        stats = torch.cuda.memory_stats(device)
        count = num_kv_blocks(total, total - free, stats["allocated_bytes.all.peak"],
                              stats["allocated_bytes.all.current"], gpu_memory_utilization,
                              kv_block_bytes(num_layers, block_size, num_kv_heads, head_dim, kv_format, track_scores),
                              cap)
        return cls(num_layers, count, block_size, num_kv_heads, head_dim, kv_format, device, track_scores)

    @property
    def fp8(self) -> bool:
        return self.kv_format == "fp8_e4m3fn"

    def _side(self, side: int):
        """K (0) or V (1) of every layer, as the kernels take it."""
        return self.kv[side].view(torch.float4_e2m1fn_x2) if self.kv_format == "fp4_e2m1" else self.kv[side]

    def layer(self, l: int):
        """(k_cache, v_cache, k_scale, v_scale) views of layer ``l`` (scales None for bf16)."""
        if self.scale is None:
            return self.kv[0, l], self.kv[1, l], None, None
        return self._side(0)[l], self._side(1)[l], self.scale[0, l], self.scale[1, l]

    def attach(self, model) -> int:
        """Assigns each layer's views to the modules that have ``k_cache``/``v_cache``, in order
        (mixed_model_runner.py:43-47); quantised pools also set ``k_scale``/``v_scale``, pools
        that track scores ``kv_scores``.
        Returns the number of layers attached."""
        layer = 0
        modules = model.modules() if hasattr(model, "modules") else model
        for module in modules:
            if hasattr(module, "k_cache") and hasattr(module, "v_cache"):
                if layer >= self.num_layers:
                    raise ValueError("more attention layers than pool layers")
                module.k_cache, module.v_cache, k_scale, v_scale = self.layer(layer)
                if self.scale is not None or hasattr(module, "k_scale"):
                    module.k_scale, module.v_scale = k_scale, v_scale
                if self.scores is not None or hasattr(module, "kv_scores"):
                    module.kv_scores = None if self.scores is None else self.scores[layer]
                layer += 1
        return layer

    # ------------------------------------------------------------- lifecycle
    def copy_blocks(self, src: list[int], dst: list[int]) -> None:
        """Copies whole blocks (codes and scales, every layer): copy-on-write of a shared block."""
        if len(src) != len(dst) or len(set(dst)) != len(dst) or set(src) & set(dst):
            raise ValueError("copy_blocks needs distinct destination blocks, disjoint from the sources")
        s = torch.as_tensor(src, dtype=torch.long, device=self.kv.device)
        d = torch.as_tensor(dst, dtype=torch.long, device=self.kv.device)
        self.kv[:, :, d] = self.kv[:, :, s]
        if self.scale is not None:
            self.scale[:, :, d] = self.scale[:, :, s]
        if self.scores is not None:
            self.scores[:, d] = self.scores[:, s]

    def reset_blocks(self, blocks: list[int]) -> None:
        """Returns blocks to the initial state (codes 0, scales 1, weights 0) before reuse."""
        b = torch.as_tensor(blocks, dtype=torch.long, device=self.kv.device)
        self.kv[:, :, b] = 0
        if self.scale is not None:
            self.scale[:, :, b] = 1.0 if self.fp8 else 127
        if self.scores is not None:
            self.scores[:, b] = 0.0

    def snapshot(self, blocks: list[int]) -> dict:
        """Host copy of whole blocks, codes, scales and accumulated weights (the geometry-aware
        form of diagnostics/online_token_replay/tensors.py:11-35)."""
        b = torch.as_tensor(blocks, dtype=torch.long, device=self.kv.device)
        image = {"block_ids": list(blocks), "kv_format": self.kv_format,
                "kv": self.kv[:, :, b].cpu(), "scale": None if self.scale is None else self.scale[:, :, b].cpu(),
                "pool_shape": list(self.kv.shape)}
        if self.scores is not None:
            image["scores"] = self.scores[:, b].cpu()
        return image

    def restore(self, image: dict) -> None:
        if image["kv_format"] != self.kv_format or image["pool_shape"] != list(self.kv.shape):
            raise ValueError("snapshot geometry or format differs from this pool")
        b = torch.as_tensor(image["block_ids"], dtype=torch.long, device=self.kv.device)
        self.kv[:, :, b] = image["kv"].to(self.kv.device)
        if self.scale is not None:
            self.scale[:, :, b] = image["scale"].to(self.kv.device)
        if self.scores is not None:  # an image of a pool without weights: they start from zero
            self.scores[:, b] = image["scores"].to(self.kv.device) if "scores" in image else 0.0

    # -------------------------------------------------------------- contents
    def read(self, l: int, slot_mapping: torch.Tensor):
        """(k, v) of layer ``l``'s tokens at the given slots as bf16 ``[N, kv_heads, head_dim]``
        (``load_kvcache``), e.g. to move them to a pool of another format."""
        k_cache, v_cache, k_scale, v_scale = self.layer(l)
        return load_kvcache(k_cache, v_cache, slot_mapping, k_scale, v_scale)

    def evict(self, lens: torch.Tensor, tables: torch.Tensor, budget: int, recent: int):
        """Cuts rows of more than ``budget`` tokens back to it in every layer (``evict_kv``); returns
        ``(new_lens, kept)``.  The caller then frees the pages past the new lengths."""
        if self.scores is None:
            raise RuntimeError("evict needs a pool with track_scores")
        k_scale, v_scale = (None, None) if self.scale is None else (self.scale[0], self.scale[1])
        return evict_kv(self._side(0), self._side(1), self.scores, lens, tables, budget, recent, k_scale, v_scale)
