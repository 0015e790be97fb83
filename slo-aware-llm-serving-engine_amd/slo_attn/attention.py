"""Drop-in ``Attention`` module and ``store_kvcache`` for the nano-vLLM engine.

Mirrors nanovllm/layers/attention.py:33-79: same constructor, attributes
(``num_heads``, ``head_dim``, ``scale``, ``num_kv_heads``, ``k_cache``,
``v_cache``) and ``forward(q, k, v)`` dispatch on the global ``Context``:

* ``context.mixed`` set -> ``forward_mixed`` (one KV write + one ragged launch);
* V0 prefill -> KV write, then causal varlen attention over the cache when
  ``block_tables`` is given (prefix cache), else over the contiguous new K/V;
* V0 decode -> KV write, then paged decode; returns ``[B, 1, Hq, D]`` like
  flash_attn_with_kvcache on ``q.unsqueeze(1)``.

Optional ``k_scale`` / ``v_scale`` attributes (fp32
``[num_blocks, block_size, num_kv_heads]``) select the E4M3FN pool when the
runner assigns uint8 / float8_e4m3fn ``k_cache`` / ``v_cache`` views; with
float4_e2m1fn_x2 views they are the E8M0 scales of a 4-bit pool (``KVPool``
allocates either).  An optional ``kv_scores`` attribute (fp32 ``[num_blocks,
num_kv_heads, block_size]``) has every step add its attention weights to the
scores of the cached tokens (``accumulate_attention``, from the pool's keys).
Prompts that come without block tables are whole: the slots that their tokens
were written to say which pages they have.
``forward(q, k, v, kv_stored=True)`` skips the KV write, for callers whose
``qk_norm_rope_store`` already wrote this step's K/V into the pool.
``Attention(..., window=W, sinks=S)`` is a layer with a sliding window: a query
sees the W newest tokens up to its own and the row's first S.  Its KV write is a
launch of its own, and it takes no ``kv_scores``.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib
from .context import get_context
from .mixed_attention import forward_mixed
from .ops import accumulate_attention, check_store, foldable, folds_alone, is_fp4, paged_attention, store_kvcache

__all__ = ["Attention", "store_kvcache"]


def _stored(*args):
    """store_fn for a step whose K/V are already in the pool."""


def _pages_of_slots(slots: torch.Tensor, cu_k: torch.Tensor, max_k: int, block_size: int) -> torch.Tensor:
    """Block tables int32 ``[rows, pages of max_k]``, -1 padded, of cold prefill rows.

    Token j of row r went to ``slots[cu_k[r] + j]``, and every ``block_size``-th
    token begins a page.  Without ``max_k`` the slots bound the rows.
    """
    if not slots.numel():
        return torch.full((cu_k.numel() - 1, 1), -1, dtype=torch.int32, device=cu_k.device)
    first = torch.arange(0, max_k if max_k > 0 else slots.numel(), block_size, dtype=cu_k.dtype, device=cu_k.device) + cu_k[:-1, None]
    slot = slots[first.clamp(max=slots.numel() - 1)]
    return torch.where((first < cu_k[1:, None]) & (slot >= 0), slot // block_size, -1)


class Attention(nn.Module):

    def __init__(self, num_heads, head_dim, scale, num_kv_heads, window=0, sinks=0):
        super().__init__()
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError("window must be positive (0 without sinks: no window) and sinks not negative")
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])
        self.k_scale = self.v_scale = None
        self.kv_scores = None
        self.window, self.sinks = window, sinks

    def _scales(self):
        return () if self.k_scale is None else (self.k_scale, self.v_scale)

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_stored: bool = False):
        context = get_context()
        k_cache, v_cache = self.k_cache, self.v_cache
        span = dict(window=self.window, sinks=self.sinks)
        if self.window and self.kv_scores is not None:
            raise ValueError("a layer with a window takes no kv_scores: attach a pool without track_scores")
        if context.mixed is not None:
            o = forward_mixed(q, k, v, k_cache, v_cache, context, self.scale,
                              _stored if kv_stored else store_kvcache, self.k_scale, self.v_scale, **span)
            if self.kv_scores is not None:
                meta = context.mixed
                self._weigh(q, num_decode=meta.num_decode, decode_lens=meta.decode_lens, decode_tables=meta.decode_tables,
                            num_prefill=meta.prefill_cu_q.numel() - 1 if meta.num_prefill_tokens else 0,
                            prefill_cu_q=meta.prefill_cu_q, prefill_cu_k=meta.prefill_cu_k, max_q=meta.max_q,
                            max_k=meta.max_k, prefill_tables=meta.prefill_tables, slots=context.slot_mapping)
            return o
        have_cache = bool(k_cache.numel() and v_cache.numel())
        # The pool is written inside the attention launch (same result, one
        # launch less) in decode steps, also from views of the QKV projection
        # and into E4M3FN pools (at most 8 query heads per kv head).  us a layer
        # against the store kernel and a launch: 16 rows of 64-1,024 tokens 18.1
        # -> 16.8, 64 rows of 512-4,096 125.6 -> 124.2; E4M3FN, both with the
        # direct kernel, 40 rows of 256-4,096 51.3 -> 49.2, 4 rows of 20-128
        # 7.5 -> 6.3.  So do cold prefill steps (no block tables), whose items
        # write their own tokens.  A prefill step that reads the pool hands over
        # contiguous bf16 rows only; otherwise the store kernel runs first.
        paged = context.is_prefill and context.block_tables is not None
        fold = have_cache and not kv_stored and not self.window and (
            (self.k_scale is None and not is_fp4(k_cache) and foldable(k, v))
            or (not paged and folds_alone(q, k, v, k_cache, self.k_scale)))
        if fold:
            check_store(k, v, k_cache, v_cache, context.slot_mapping, *self._scales())
        elif have_cache and not kv_stored:
            store_kvcache(k, v, k_cache, v_cache, context.slot_mapping, *self._scales())
        store = dict(store_slot_mapping=context.slot_mapping, new_k=k, new_v=v) if fold else {}
        if context.is_prefill:
            rows = context.cu_seqlens_q.numel() - 1
            pool = paged or fold
            o = paged_attention(
                q, k_cache if pool else None, v_cache if pool else None, self.scale,
                num_kv_heads=self.num_kv_heads, k_scale=self.k_scale if pool else None,
                v_scale=self.v_scale if pool else None, num_prefill=rows,
                prefill_cu_q=context.cu_seqlens_q, prefill_cu_k=context.cu_seqlens_k,
                max_q=context.max_seqlen_q, max_k=context.max_seqlen_k,
                prefill_tables=context.block_tables, k=None if paged else k, v=None if paged else v,
                phases=_lib.PHASE_ALL if paged else _lib.PHASE_ALL | _lib.NEW_ROWS_STRIDED, **store, **span)
            if self.kv_scores is not None and have_cache:
                self._weigh(q, num_prefill=rows, prefill_cu_q=context.cu_seqlens_q, prefill_cu_k=context.cu_seqlens_k,
                            max_q=context.max_seqlen_q, max_k=context.max_seqlen_k, prefill_tables=context.block_tables,
                            slots=context.slot_mapping)
            return o
        o = paged_attention(
            q, k_cache, v_cache, self.scale, num_kv_heads=self.num_kv_heads,
            k_scale=self.k_scale, v_scale=self.v_scale, num_decode=q.shape[0],
            decode_lens=context.context_lens, decode_tables=context.block_tables,
            phases=_lib.PHASE_ALL | _lib.NEW_ROWS_STRIDED, **store, **span)
        if self.kv_scores is not None:
            self._weigh(q, num_decode=q.shape[0], decode_lens=context.context_lens, decode_tables=context.block_tables)
        return o.unsqueeze(1)

    def _weigh(self, q, slots=None, **rows):
        """The step's attention weights into ``kv_scores``; ``slots`` are the new tokens', decode rows first."""
        if rows.get("num_prefill") and rows["prefill_tables"] is None and slots is not None:
            rows["prefill_tables"] = _pages_of_slots(slots[rows.get("num_decode", 0):], rows["prefill_cu_k"], rows["max_k"],
                                                     self.kv_scores.shape[2])
        accumulate_attention(q, self.k_cache, self.kv_scores, self.scale, num_kv_heads=self.num_kv_heads,
                             k_scale=self.k_scale, **rows)
