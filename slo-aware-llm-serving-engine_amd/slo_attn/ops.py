"""Host wrappers around the C-ABI: argument checks, workspace, stream plumbing.

Every function here launches hand-written HIP kernels through libslo_attn.so on
the current PyTorch stream.  Nothing allocates device memory except the output
tensor and the one-time, per-device workspace (grown outside graph capture), so
calls may be captured into a HIP graph once the workspace is reserved.
There is no CPU path: CPU tensors are rejected.
"""
from __future__ import annotations

import contextlib
import ctypes
import threading

import torch

from . import _lib

_FP4_DTYPE = getattr(torch, "float4_e2m1fn_x2", None)
_FP32 = (torch.float32,)
_E8M0_DTYPES = (torch.uint8,) + ((torch.float8_e8m0fnu,) if hasattr(torch, "float8_e8m0fnu") else ())
_FP8_DTYPES = (torch.uint8,) + ((torch.float8_e4m3fn,) if hasattr(torch, "float8_e4m3fn") else ())


def kv_dtype_code(cache: torch.Tensor) -> int:
    if cache.dtype == torch.bfloat16:
        return _lib.KV_BF16
    if cache.dtype in _FP8_DTYPES:
        return _lib.KV_FP8_E4M3FN
    if cache.dtype == _FP4_DTYPE:
        return _lib.KV_FP4_E2M1
    raise TypeError(f"KV cache dtype {cache.dtype} is not bf16, E4M3FN bytes or float4_e2m1fn_x2")


def is_fp4(cache: torch.Tensor | None) -> bool:
    """Whether a pool view is a 4-bit one (``torch.float4_e2m1fn_x2``: two E2M1 codes a byte)."""
    return cache is not None and _FP4_DTYPE is not None and cache.dtype == _FP4_DTYPE


def _pool_geometry(k_cache, k_scale, v_cache=None, v_scale=None, want_v=True):
    """Checks a layer's pool views and returns ``(code, blocks, block_size, kv_heads, head_dim)``.

    bf16 and E4M3FN pools are ``[blocks, block_size, kv_heads, head_dim]`` with
    fp32 scales ``[blocks, block_size, kv_heads]`` (E4M3FN); 4-bit pools
    ``[blocks, kv_heads, block_size, head_dim / 2]`` with E8M0 scales
    ``[blocks, kv_heads, block_size, head_dim / 32]``.
    """
    code = kv_dtype_code(k_cache)
    shape = k_cache.shape
    if len(shape) != 4 or not k_cache.is_contiguous():
        raise ValueError("KV pool views must be contiguous and 4-dimensional")
    if want_v:
        if kv_dtype_code(v_cache) != code:
            raise TypeError("k_cache and v_cache formats differ")
        if v_cache.shape != shape or not v_cache.is_contiguous():
            raise ValueError("k_cache and v_cache must be contiguous and of one shape")
    if code == _lib.KV_FP4_E2M1:
        blocks, heads, block, d = shape
        d *= 2
        want, dtypes = (blocks, heads, block, d // _lib.FP4_GROUP), _E8M0_DTYPES
    else:
        blocks, block, heads, d = shape
        want, dtypes = (blocks, block, heads), _FP32
    if code != _lib.KV_BF16:
        for sc in (k_scale, v_scale) if want_v else (k_scale,):
            if sc is None:
                raise ValueError("a quantised pool needs its scales")
            if sc.dtype not in dtypes or sc.shape != want or not sc.is_contiguous():
                kind = "E8M0" if code == _lib.KV_FP4_E2M1 else "fp32"
                raise ValueError(f"scale pools must be contiguous {kind} {list(want)}")
    return code, blocks, block, heads, d


def _check_scores(kv_scores, blocks, heads, block, layers=()):
    if kv_scores.dtype != torch.float32:
        raise TypeError("kv_scores must be fp32")
    if kv_scores.shape != (*layers, blocks, heads, block) or not kv_scores.is_contiguous():
        raise ValueError("kv_scores must be contiguous fp32 [num_blocks, num_kv_heads, block_size]")


def _require_gpu(*tensors) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("slo_attn kernels need GPU tensors; there is no CPU fallback")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError(f"tensors on different devices: {device} vs {t.device}")
    return device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _one_device(first: torch.Tensor, *others) -> int:
    """The index of the GPU that holds all tensors (None: left out)."""
    device = first.device
    if device.type != "cuda":
        raise RuntimeError("slo_attn kernels need GPU tensors; there is no CPU fallback")
    for t in others:
        if t is not None and t.device != device:
            if t.device.type != "cuda":
                raise RuntimeError("slo_attn kernels need GPU tensors; there is no CPU fallback")
            raise RuntimeError(f"tensors on different devices: {device} vs {t.device}")
    return device.index


def _launch(index: int, what: str, *args) -> None:
    """Calls an entry point on the current stream of GPU ``index``, which need not be the current one."""
    lib = _lib.load()
    with contextlib.nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index):
        rc = getattr(lib, what)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _int32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() == 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t


# ------------------------------------------------------------------ KV write
def check_store(key, value, k_cache, v_cache, slot_mapping, k_scale=None, v_scale=None):
    """The store's argument checks (nanovllm/layers/attention.py:36-39 and the
    formats); returns ``(device, kv_dtype code)``."""
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    if is_fp4(k_cache):
        index, _ = _check_store_fp4(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
        return torch.device("cuda", index), _lib.KV_FP4_E2M1
    # Same stride contract as the reference store (attention.py:36-39).
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    device = _require_gpu(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError("key/value must be bf16")
    if value.shape != key.shape:
        raise ValueError("key/value shapes differ")
    code = kv_dtype_code(k_cache)
    if kv_dtype_code(v_cache) != code:
        raise TypeError("k_cache and v_cache formats differ")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV pool views must be contiguous")
    num_slots = k_cache.shape[0] * k_cache.shape[1]
    if code == _lib.KV_FP8_E4M3FN:
        if k_scale is None or v_scale is None:
            raise ValueError("an E4M3FN pool needs k_scale and v_scale")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or not s.is_contiguous() or s.numel() != num_slots * num_heads:
                raise ValueError("scale pools must be contiguous fp32 [num_blocks, block_size, num_kv_heads]")
    _int32(slot_mapping, "slot_mapping")
    return device, code


def _check_store_fp4(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale):
    """``check_store`` for a 4-bit pool; returns ``(device index, its geometry)``."""
    N, num_heads, head_dim = shape = key.shape
    ks, vs = key.stride(), value.stride()
    assert ks[2] == 1 and vs[2] == 1
    assert ks[1] == head_dim and vs[1] == head_dim
    assert slot_mapping.numel() == N
    index = _one_device(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError("key/value must be bf16")
    if value.shape != shape:
        raise ValueError("key/value shapes differ")
    geometry = _pool_geometry(k_cache, k_scale, v_cache, v_scale)
    if geometry[3] != num_heads or geometry[4] != head_dim:
        raise ValueError("KV pool must be [num_blocks, num_kv_heads, block_size, head_dim / 2]")
    _int32(slot_mapping, "slot_mapping")
    return index, geometry


def foldable(key: torch.Tensor, value: torch.Tensor) -> bool:
    """Whether the attention launch can carry the KV write of these new rows:
    bf16 ``[N, num_kv_heads, head_dim]`` rows stored back to back."""
    row = key.shape[1] * key.shape[2]
    return (key.dim() == 3 and key.dtype == torch.bfloat16 and value.dtype == torch.bfloat16
            and key.stride(0) == row and value.stride(0) == row and key.stride(2) == 1 and value.stride(2) == 1
            and key.stride(1) == key.shape[2] and value.stride(1) == value.shape[2])


def foldable_strided(key: torch.Tensor, value: torch.Tensor) -> bool:
    """Whether a launch without prefill rows, or of cold prefill rows only, can
    carry the KV write of these new rows (``_lib.NEW_ROWS_STRIDED``): bf16
    ``[N, num_kv_heads, head_dim]`` rows of contiguous heads on 16-byte
    boundaries, such as the K and V views of a fused QKV projection's output."""
    if key.dim() != 3 or key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        return False
    row, d = key.shape[1] * key.shape[2], key.shape[2]
    return all(t.stride(2) == 1 and t.stride(1) == d and t.stride(0) >= row and t.stride(0) % 8 == 0
               and t.data_ptr() % 16 == 0 for t in (key, value))


def folds_alone(q: torch.Tensor, key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                k_scale: torch.Tensor | None) -> bool:
    """Whether a launch of decode rows only, or of cold prefill rows only,
    carries the KV write of ``key``/``value``: ``foldable_strided`` rows, one
    per query row, into a 4-dimensional pool view; with an E4M3FN pool at most
    8 query heads per kv head.  Everything else (keys of a whole cold row
    beside the queries of its last tokens, a pool view of merged heads, a 4-bit
    pool) keeps the store kernel's own launch, which takes it."""
    return (not is_fp4(k_cache) and key.dim() == 3 and key.shape[0] == q.shape[0] and k_cache.dim() == 4 and foldable_strided(key, value)
            and (k_scale is None or q.shape[1] <= 8 * key.shape[1]))


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  scale_floor: float = _lib.FP8_SCALE_FLOOR) -> None:
    """Slot-mapped KV write (nanovllm/layers/attention.py:33-40), bf16 or E4M3FN.

    ``key``/``value``: ``[N, num_kv_heads, head_dim]`` bf16 whose rows may be
    strided (a view of the fused QKV output).  ``k_cache``/``v_cache``:
    ``[num_blocks, block_size, num_kv_heads, head_dim]``; for E4M3FN caches
    (uint8 or float8_e4m3fn) ``k_scale``/``v_scale`` are the fp32
    ``[num_blocks, block_size, num_kv_heads]`` scale pools.  4-bit caches
    (float4_e2m1fn_x2) are ``[num_blocks, num_kv_heads, block_size,
    head_dim / 2]`` with E8M0 scales ``[num_blocks, num_kv_heads, block_size,
    head_dim / 32]`` (uint8 or float8_e8m0fnu), one per 32 channels;
    ``scale_floor`` is then a power of two.
    """
    if is_fp4(k_cache):
        index, (_, blocks, block, _, _) = _check_store_fp4(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
        N, num_heads, head_dim = key.shape
        _launch(index, "slo_store_kvcache_fp4", key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0),
                slot_mapping.data_ptr(), N, num_heads, head_dim, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), blocks, block, scale_floor)
        return
    device, code = check_store(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)
    N, num_heads, head_dim = key.shape
    num_slots = k_cache.shape[0] * k_cache.shape[1]
    lib = _lib.load()
    _lib.check(lib.slo_store_kvcache(
        _ptr(key), key.stride(0), _ptr(value), value.stride(0), _ptr(slot_mapping), N, num_heads,
        head_dim, code, _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), num_slots,
        float(scale_floor), _stream(device)), "slo_store_kvcache")


def load_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
    """Cached tokens read back: ``(k, v)``, bf16 ``[N, num_kv_heads, head_dim]`` rows of the tokens at
    ``slot_mapping`` (int32), the inverse of ``store_kvcache``.

    For moving tokens to a pool of another format or to the host.  bf16 rows
    come back as stored, 4-bit values exactly, E4M3FN values as code * scale
    rounded to bf16; a slot outside the pool gives zeros.
    """
    index = _one_device(k_cache, v_cache, slot_mapping, k_scale, v_scale)
    code, blocks, block, heads, head_dim = _pool_geometry(k_cache, k_scale, v_cache, v_scale)
    if slot_mapping.dtype != torch.int32 or slot_mapping.dim() != 1 or slot_mapping.stride(0) != 1:
        raise ValueError("slot_mapping must be a contiguous 1-dimensional int32 tensor")
    N = slot_mapping.numel()
    k = torch.empty((N, heads, head_dim), dtype=torch.bfloat16, device=k_cache.device)
    v = torch.empty_like(k)
    _launch(index, "slo_load_kvcache", k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_scale), _ptr(v_scale), code, blocks,
            block, slot_mapping.data_ptr(), N, heads, head_dim, k.data_ptr(), v.data_ptr())
    return k, v


# ------------------------------------------- fused q/k norm + RoPE + KV write
def rope_cos_sin(head_dim: int, max_position: int, base: float, device) -> torch.Tensor:
    """fp32 [max_position, head_dim] table: cos(p * inv_freq) then sin(p * inv_freq).

    The cos_sin_cache of RotaryEmbedding (nanovllm/layers/rotary_embedding.py:27-35),
    built with the same torch operations on ``device``.
    """
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float, device=device) / head_dim))
    t = torch.arange(max_position, dtype=torch.float, device=device)
    freqs = torch.einsum("i,j -> ij", t, inv_freq)
    return torch.cat((freqs.cos(), freqs.sin()), dim=-1).contiguous()


def qk_norm_rope_store(qkv: torch.Tensor, positions: torch.Tensor, q_norm_weight: torch.Tensor,
                       k_norm_weight: torch.Tensor, eps: float, cos_sin: torch.Tensor, num_heads: int,
                       num_kv_heads: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                       v_scale: torch.Tensor | None = None, head_dim: int = 128,
                       scale_floor: float = _lib.FP8_SCALE_FLOOR):
    """q_norm, k_norm, rotary_emb and the KV write of one layer in one launch.

    Covers nanovllm/models/qwen3.py:80-86 up to the attention call, and the
    store_kvcache that Attention.forward would issue (attention.py:59-66).
    ``qkv``: ``[N, (num_heads + 2*num_kv_heads) * head_dim]`` bf16 (the fused
    projection output; rows may be strided).  Returns ``(q, k, v)``: q and k
    normalised and rotated (new contiguous bf16 tensors), v a view of ``qkv``.
    The pool receives the rotated k and v at ``slot_mapping`` (bf16, or
    E4M3FN or 4 bits with ``k_scale``/``v_scale``), as ``store_kvcache`` writes
    them; into a 4-bit pool they go in a second launch.
    """
    if qkv.dim() != 2 or qkv.stride(-1) != 1:
        raise ValueError("qkv must be a [tokens, width] tensor with contiguous rows")
    N = qkv.shape[0]
    width = (num_heads + 2 * num_kv_heads) * head_dim
    if qkv.shape[1] != width:
        raise ValueError(f"qkv rows must hold {width} elements")
    device = _require_gpu(qkv, positions, q_norm_weight, k_norm_weight, cos_sin, k_cache, v_cache,
                          slot_mapping, k_scale, v_scale)
    if qkv.dtype != torch.bfloat16:
        raise TypeError("qkv must be bf16")
    if positions.dtype != torch.int64 or positions.numel() != N or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int64 [tokens] tensor")
    for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if w.dtype != torch.bfloat16 or w.numel() != head_dim or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bf16 [head_dim] tensor")
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.shape[1] != head_dim or \
            not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous fp32 [max_position, head_dim] table")
    code = kv_dtype_code(k_cache)
    if kv_dtype_code(v_cache) != code:
        raise TypeError("k_cache and v_cache formats differ")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV pool views must be contiguous")
    fp4 = code == _lib.KV_FP4_E2M1
    if fp4:
        if _pool_geometry(k_cache, k_scale, v_cache, v_scale)[3:] != (num_kv_heads, head_dim):
            raise ValueError("KV pool must be [num_blocks, num_kv_heads, block_size, head_dim / 2]")
    elif k_cache.shape[-2:] != (num_kv_heads, head_dim) or v_cache.shape != k_cache.shape:
        raise ValueError("KV pool must be [num_blocks, block_size, num_kv_heads, head_dim]")
    # A pool of no slots: the fused kernel writes q and k only.
    num_slots = 0 if fp4 else k_cache.shape[0] * k_cache.shape[1]
    if code == _lib.KV_FP8_E4M3FN:
        if k_scale is None or v_scale is None:
            raise ValueError("an E4M3FN pool needs k_scale and v_scale")
        for sc in (k_scale, v_scale):
            if sc.dtype != torch.float32 or not sc.is_contiguous() or sc.numel() != num_slots * num_kv_heads:
                raise ValueError("scale pools must be contiguous fp32 [num_blocks, block_size, num_kv_heads]")
    _int32(slot_mapping, "slot_mapping")
    if slot_mapping.numel() != N:
        raise ValueError("slot_mapping must hold one slot per token")
    q = torch.empty((N, num_heads, head_dim), dtype=torch.bfloat16, device=qkv.device)
    k = torch.empty((N, num_kv_heads, head_dim), dtype=torch.bfloat16, device=qkv.device)
    _lib.check(_lib.load().slo_qk_norm_rope_store(
        _ptr(qkv), qkv.stride(0), _ptr(positions), N, num_heads, num_kv_heads, head_dim, _ptr(q_norm_weight),
        _ptr(k_norm_weight), float(eps), _ptr(cos_sin), cos_sin.shape[0], _ptr(q), _ptr(k), _ptr(slot_mapping),
        _lib.KV_BF16 if fp4 else code, _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), num_slots,
        float(scale_floor), _stream(device)), "slo_qk_norm_rope_store")
    v = qkv[:, (num_heads + num_kv_heads) * head_dim:].view(N, num_kv_heads, head_dim)
    if fp4:
        store_kvcache(k, v, k_cache, v_cache, slot_mapping, k_scale, v_scale, scale_floor)
    return q, k, v


# ------------------------------------------------------ LM head + greedy argmax
_keys: dict[int, torch.Tensor] = {}
LM_HEAD_MAX_ROWS = 128


def lm_head_argmax(hidden: torch.Tensor, weight: torch.Tensor, return_logits: bool = False):
    """Greedy next tokens of the sampled rows: argmax_v bf16(hidden[r] . weight[v]).

    compute_logits + argmax of run_mixed (nanovllm/engine/mixed_model_runner.py:
    115-126, nanovllm/layers/embed_head.py:56-66) in one pass over the weight.
    ``hidden``: ``[rows, hidden_size]`` bf16 (the already-selected sampled rows,
    at most 128); ``weight``: ``[vocab, hidden_size]`` bf16.  Returns int64
    ``[rows]`` tokens (ties: the smallest index), and the bf16 logits
    ``[rows, vocab]`` as well when ``return_logits``.
    """
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError("hidden must be [rows, hidden_size] and weight [vocab, hidden_size]")
    device = _require_gpu(hidden, weight)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("hidden and weight must be bf16")
    if hidden.stride(-1) != 1 or weight.stride(-1) != 1:
        raise ValueError("hidden and weight rows must be contiguous")
    rows, vocab = hidden.shape[0], weight.shape[0]
    if rows > LM_HEAD_MAX_ROWS:
        raise ValueError(f"at most {LM_HEAD_MAX_ROWS} sampled rows per call")
    index = device.index if device.index is not None else torch.cuda.current_device()
    keys = _keys.get(index)
    if keys is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call lm_head_argmax once before graph capture")
        keys = torch.zeros(LM_HEAD_MAX_ROWS, dtype=torch.int64, device=device)
        _keys[index] = keys
    tokens = torch.empty(rows, dtype=torch.int64, device=device)
    logits = torch.empty(rows, vocab, dtype=torch.bfloat16, device=device) if return_logits else None
    _lib.check(_lib.load().slo_lm_head_argmax(
        _ptr(hidden), hidden.stride(0), rows, _ptr(weight), weight.stride(0), vocab, hidden.shape[1], _ptr(logits),
        vocab, _ptr(keys), _ptr(tokens), _stream(device)), "slo_lm_head_argmax")
    return (tokens, logits) if return_logits else tokens


# ---------------------------------------------------------------- workspace
_ws_lock = threading.Lock()
_workspaces: dict[int, torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Per-device zero-initialised workspace of at least ``nbytes`` bytes.

    The kernels leave the control words and split-K tickets at zero when they
    finish, so the buffer is zero-filled only when it is (re)allocated.
    Growing is refused while a graph is being captured.
    """
    index = device.index if device.index is not None else torch.cuda.current_device()
    with _ws_lock:
        ws = _workspaces.get(index)
        if ws is not None and ws.numel() >= nbytes:
            return ws
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("attention workspace must be reserved before graph capture "
                               "(call reserve_workspace)")
        size = max(nbytes, int((ws.numel() if ws is not None else 0) * 1.5), 1 << 20)
        ws = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", index))
        _workspaces[index] = ws
        return ws


def check_workspaces() -> None:
    """Raise if any device's attention workspace is not in the state every
    launch leaves it in (work-list counters and split-K tickets zero), or if a
    split-K merge gave up waiting since the last check (its decode outputs were
    not written).  Synchronises the current stream of each device; call it
    outside graph capture, e.g. every few hundred steps of a serving loop."""
    for index, ws in list(_workspaces.items()):
        device = torch.device("cuda", index)
        _lib.check(_lib.load().slo_attention_workspace_check(ws.data_ptr(), ws.numel(), None, _stream(device)),
                   "slo_attention_workspace_check")


def workspace_events(device) -> dict:
    """Reads and clears the attention workspace's event counters on ``device``
    (after checking its zero invariants): ``merges_gave_up`` (split-K merge
    tasks that stopped waiting) and ``split_prefill_merges`` (split prefill
    item pairs merged).  Raises like ``check_workspaces`` when a merge gave up.
    Synchronises; a diagnostic for tests and tuning."""
    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    ws = _workspaces.get(index)
    if ws is None:
        return {"merges_gave_up": 0, "split_prefill_merges": 0}
    ev = (ctypes.c_uint32 * 4)()
    _lib.check(_lib.load().slo_attention_workspace_check(ws.data_ptr(), ws.numel(), ev, _stream(device)),
               "slo_attention_workspace_check")
    return {"merges_gave_up": int(ev[0]), "split_prefill_merges": int(ev[1])}


def reserve_workspace(device, max_decode_rows: int, max_decode_len: int, num_heads: int,
                      num_kv_heads: int, head_dim: int) -> torch.Tensor:
    nbytes = _lib.workspace_bytes(max_decode_rows, max_decode_len, num_heads, num_kv_heads, head_dim)
    return workspace(torch.device(device), nbytes)


# ---------------------------------------------------------------- attention
def _row_args(T, num_decode, decode_lens, decode_tables, num_prefill, cu_q, cu_k, max_q, max_k, tables, phases):
    """Checks the rows of the asked phases, all read through block tables, and returns their fields of
    ``PagedAttentionArgs``: those of the decode rows, then those of the prefill rows."""
    if not 0 <= num_decode <= T:
        raise ValueError("num_decode must be from 0 to the number of query rows")
    decode, prefill = (num_decode, None, None, 0, 0), (0, None, None, 0, 0, None, 0, 0)
    if num_prefill and cu_q is not None:  # where the prefill rows end matters in either phase
        _int32(cu_q, "cu_seqlens_q")
        if cu_q.numel() < num_prefill + 1:
            raise ValueError("cu_seqlens shorter than num_prefill + 1")
        prefill = num_prefill, cu_q.data_ptr(), *prefill[2:]
    if num_decode and phases & _lib.PHASE_DECODE:
        _int32(decode_lens, "decode_lens")
        _int32(decode_tables, "decode_tables")
        if decode_tables.dim() != 2 or decode_tables.stride(1) != 1:
            raise ValueError("decode_tables must be a row-major [rows, width] int32 tensor")
        rows, width = decode_tables.shape
        if decode_lens.numel() < num_decode or rows < num_decode:
            raise ValueError("decode metadata has fewer rows than num_decode")
        decode = num_decode, decode_lens.data_ptr(), decode_tables.data_ptr(), decode_tables.stride(0), width
    if num_prefill and phases & _lib.PHASE_PREFILL:
        _int32(cu_q, "cu_seqlens_q")
        _int32(cu_k, "cu_seqlens_k")
        _int32(tables, "block_tables")
        if cu_q.numel() < num_prefill + 1 or cu_k.numel() < num_prefill + 1:
            raise ValueError("cu_seqlens shorter than num_prefill + 1")
        if tables.dim() != 2 or tables.stride(1) != 1 or tables.shape[0] < num_prefill:
            raise ValueError("block_tables must be a row-major [rows, width] int32 tensor")
        prefill = (num_prefill, cu_q.data_ptr(), cu_k.data_ptr(), int(max_q), int(max_k), tables.data_ptr(), tables.stride(0),
                   tables.shape[1])
    return decode, prefill


_NO_ROWS, _NO_STORE = (None, 0, None, 0, 0), (None, None, 0, None, 0, 0, 0.0)


def _pool_call(what, extra, index, device, q, out, k_cache, v_cache, k_scale, v_scale, geometry, rows, scale, phases):
    """Calls ``what`` over a pool with a workspace of the call's own, from torch's allocator: calls on several streams,
    and graphs captured apart, do not share one, and it need not be cleared."""
    code, blocks, block, heads, head_dim = geometry
    T, num_heads, _ = q.shape
    decode, prefill = rows
    fields = (q.data_ptr(), q.stride(0) if T > 1 else num_heads * head_dim, _ptr(out) or 0,
              0 if out is None else out.stride(0) if T > 1 else num_heads * head_dim, T, k_cache.data_ptr(), _ptr(v_cache) or 0,
              _ptr(k_scale) or 0, _ptr(v_scale) or 0, code, blocks, block, *(x or 0 for x in decode), *(x or 0 for x in prefill),
              0, 0, 0, 0, 0, num_heads, heads, head_dim, scale)
    args = _lib.pack_attention_args(*fields, 0, 0, phases, 0, 0, 0, 0, 0, 0, 0.0)
    need = _workspace_need(args, what, T, num_heads, heads, code, block, phases, decode[0], decode[4], prefill[0], prefill[3],
                           prefill[4], prefill[7])
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        args = _lib.pack_attention_args(*fields, ws.data_ptr(), need, phases, 0, 0, 0, 0, 0, 0, 0.0)
    _launch(index, what, args, *extra)


_sizes: dict[tuple, int] = {}  # workspace bytes by entry point and sizes


def _workspace_need(args, *key) -> int:
    what = key[0]
    need = _sizes.get(key)
    if need is None:
        size = ctypes.c_size_t(0)
        _lib.check(getattr(_lib.load(), what + "_workspace_bytes")(args, ctypes.byref(size)), what)
        if len(_sizes) >= 4096:
            _sizes.clear()
        need = _sizes[key] = size.value
    return need


def accumulate_attention(q: torch.Tensor, k_cache: torch.Tensor, kv_scores: torch.Tensor, softmax_scale: float, *,
                         num_kv_heads: int, k_scale: torch.Tensor | None = None, num_decode: int = 0,
                         decode_lens: torch.Tensor | None = None, decode_tables: torch.Tensor | None = None,
                         num_prefill: int = 0, prefill_cu_q: torch.Tensor | None = None,
                         prefill_cu_k: torch.Tensor | None = None, max_q: int = 0, max_k: int = 0,
                         prefill_tables: torch.Tensor | None = None, phases: int = _lib.PHASE_ALL) -> None:
    """Adds the attention weights of a step's queries to their keys' scores.

    The rows are ``paged_attention``'s, over a bf16, E4M3FN or 4-bit pool, all
    read through block tables.  ``kv_scores`` (fp32 ``[num_blocks,
    num_kv_heads, block_size]``) gains, for every cached key of a row, the sum
    over the row's queries and over the query heads of the kv head of their
    softmax weights; the row's new tokens (the last one of a decode row, the
    last ``cu_q[r+1] - cu_q[r]`` of a prefill row) start from that sum, whatever
    their slots held.  A cached prefix that was never weighed has to be zero
    (``KVPool.reset_blocks``).  Rows of one call may share old pages: each adds
    its weights, in an order that is not fixed.  ``max_q`` and ``max_k`` only
    size the launches; given, they keep them small.  ``evict_kv`` reads the scores.
    """
    index, geometry = _check_query(q, num_kv_heads, k_cache, k_scale, None, None, False, kv_scores, decode_lens, decode_tables,
                                   prefill_cu_q, prefill_cu_k, prefill_tables)
    _check_scores(kv_scores, geometry[1], num_kv_heads, geometry[2])
    phases &= _lib.PHASE_ALL
    if num_prefill and phases & _lib.PHASE_PREFILL and prefill_tables is None:
        raise ValueError("accumulate_attention reads prefill rows through block tables")
    rows = _row_args(q.shape[0], num_decode, decode_lens, decode_tables, num_prefill, prefill_cu_q, prefill_cu_k, max_q, max_k,
                     prefill_tables, phases)
    _pool_call("slo_accumulate_attention", (kv_scores.data_ptr(),), index, q.device, q, None, k_cache, None, k_scale, None,
               geometry, rows, float(softmax_scale), phases)


def _check_query(q, num_kv_heads, k_cache, k_scale, v_cache, v_scale, want_v, *others):
    """Checks q against a pool; returns ``(device index, the pool's geometry)``."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, num_heads, head_dim]")
    index = _one_device(q, k_cache, k_scale, v_cache, v_scale, *others)
    if q.dtype != torch.bfloat16:
        raise TypeError("q must be bf16")
    stride, head_dim = q.stride(), q.shape[2]
    if stride[2] != 1 or stride[1] != head_dim:
        raise ValueError("q rows must hold contiguous heads")
    geometry = _pool_geometry(k_cache, k_scale, v_cache, v_scale, want_v)
    if geometry[3] != num_kv_heads or geometry[4] != head_dim:
        raise ValueError(f"KV pool holds {geometry[3]} kv heads of {geometry[4]}, not {num_kv_heads} of {head_dim}")
    return index, geometry


def evict_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scores: torch.Tensor, lens: torch.Tensor,
             tables: torch.Tensor, budget: int, recent: int, k_scale: torch.Tensor | None = None,
             v_scale: torch.Tensor | None = None):
    """Cuts rows of more than ``budget`` cached tokens back to it; returns ``(new_lens, kept)``.

    Such a row keeps, for every kv head by itself, its newest ``recent`` tokens
    and the ``budget - recent`` others with the largest ``kv_scores`` (ties: the
    lowest position; NaN below every number).  They are moved, in position
    order, with their scales and scores, to the row's first ``budget`` places,
    so the row is from then on one of ``budget`` tokens whose further pages can
    be freed; the scores of the places given up become zero.  Rotated keys keep
    their positions: new tokens go to the next free place of the row but are
    rotated by their own position in the text.

    ``lens`` int32 ``[rows]`` and ``tables`` int32 ``[rows, width]`` describe the
    rows; no two may share a page.  With a leading layer dimension on the pools,
    the scales and the scores (``pool.kv[0]`` of every layer), all layers are cut
    by one call, each by its own scores.  ``new_lens`` is int32 ``[rows]``,
    ``kept`` the kept positions, int32 ``[(layers,) rows, num_kv_heads, budget]``,
    -1 past a row that is shorter.
    """
    index = _one_device(k_cache, v_cache, kv_scores, lens, tables, k_scale, v_scale)
    layered = k_cache.dim() == 5
    if layered and (v_cache.shape != k_cache.shape or kv_scores.shape[:1] != k_cache.shape[:1]
                    or any(s is not None and s.shape[:1] != k_cache.shape[:1] for s in (k_scale, v_scale))
                    or any(t is not None and not t.is_contiguous() for t in (k_cache, v_cache, kv_scores, k_scale, v_scale))):
        raise ValueError("pools, scales and scores of several layers must be contiguous, with one leading layer dimension")
    layers = k_cache.shape[0] if layered else 1
    one = [t if t is None or not layered else t[0] for t in (k_cache, k_scale, v_cache, v_scale)]
    code, blocks, block, heads, head_dim = _pool_geometry(*one)
    _check_scores(kv_scores, blocks, heads, block, (layers,) if layered else ())
    _int32(lens, "lens")
    _int32(tables, "tables")
    if lens.dim() != 1 or tables.dim() != 2 or tables.stride(1) != 1 or tables.shape[0] != lens.numel():
        raise ValueError("lens must be [rows] and tables a row-major [rows, width] int32 tensor")
    rows, budget, recent = lens.numel(), int(budget), int(recent)
    if budget <= 0 or not 0 <= recent <= budget:
        raise ValueError("budget must be positive and recent from 0 to budget")
    new_lens = torch.empty(rows, dtype=torch.int32, device=lens.device)
    kept = torch.empty((*((layers,) if layered else ()), rows, heads, budget), dtype=torch.int32, device=lens.device)
    args = _lib.EvictKvArgs(
        _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(kv_scores), code, layers, blocks, block, heads,
        head_dim, rows, _ptr(lens), _ptr(tables), tables.stride(0), tables.shape[1], budget, recent, _ptr(new_lens),
        _ptr(kept))
    _launch(index, "slo_evict_kv", ctypes.byref(args))
    return new_lens, kept


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor | None, v_cache: torch.Tensor | None,
                    softmax_scale: float, *, num_kv_heads: int,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    num_decode: int = 0, decode_lens: torch.Tensor | None = None,
                    decode_tables: torch.Tensor | None = None,
                    num_prefill: int = 0, prefill_cu_q: torch.Tensor | None = None,
                    prefill_cu_k: torch.Tensor | None = None, max_q: int = 0, max_k: int = 0,
                    prefill_tables: torch.Tensor | None = None,
                    k: torch.Tensor | None = None, v: torch.Tensor | None = None,
                    phases: int = _lib.PHASE_ALL, out: torch.Tensor | None = None,
                    store_slot_mapping: torch.Tensor | None = None, new_k: torch.Tensor | None = None,
                    new_v: torch.Tensor | None = None, noalloc: bool = False,
                    store_scale_floor: float = _lib.FP8_SCALE_FLOOR) -> torch.Tensor:
    """One ragged launch: decode rows ``q[:num_decode]``, then prefill rows.

    Decode row b attends to ``decode_lens[b]`` cached tokens through
    ``decode_tables[b]``.  Prefill row r owns query rows
    ``num_decode + [cu_q[r], cu_q[r+1])`` and attends causally, bottom-right
    aligned, to ``cu_k[r+1]-cu_k[r]`` keys from the pool (``prefill_tables``)
    or, with ``prefill_tables=None``, from the contiguous ``k``/``v`` rows
    starting at ``cu_k[r]``.  Returns ``out`` ``[q rows, num_heads, head_dim]``.

    With ``store_slot_mapping``, the same launch also writes ``new_k``/``new_v``
    (one row per query row: decode tokens, then prefill tokens) to their slots,
    the store of forward_mixed folded in, and reads the step's new tokens from
    those rows; the result is the separate store followed by the launch, bit
    for bit.  With an E4M3FN pool the write is ``store_kvcache``'s quantising
    store (``store_scale_floor``), the new tokens are read as its codes and
    scales, and at most 8 query heads may share a kv head.

    A 4-bit pool (``store_kvcache``) is read by kernels of its own, one launch
    for the decode rows and one for the prefill rows (and one that joins the
    parts of long rows); ``store_slot_mapping`` then stores first.  Prefill rows
    without tables read no pool and run as with any other.  ``noalloc`` is
    refused.  ``max_q`` and ``max_k`` may be left out with any pool: results do
    not depend on them.

    ``noalloc=True`` launches through ``slo_paged_attention_noalloc``, which
    uses the library's static per-GPU scratch instead of this module's
    workspace (pass ``out`` as well and nothing is allocated).
    """
    if is_fp4(k_cache):
        return _paged_attention_fp4(q, k_cache, v_cache, softmax_scale, num_kv_heads, k_scale, v_scale, num_decode, decode_lens,
                                    decode_tables, num_prefill, prefill_cu_q, prefill_cu_k, max_q, max_k, prefill_tables, k, v,
                                    phases, out, store_slot_mapping, new_k, new_v, noalloc, store_scale_floor)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, num_heads, head_dim]")
    T, num_heads, head_dim = q.shape
    device = _require_gpu(q, k_cache, v_cache, k_scale, v_scale, decode_lens, decode_tables,
                          prefill_cu_q, prefill_cu_k, prefill_tables, k, v, out)
    if q.dtype != torch.bfloat16:
        raise TypeError("q must be bf16")
    if q.stride(-1) != 1 or q.stride(1) != head_dim:
        raise ValueError("q rows must hold contiguous heads")
    if out is None:
        out = torch.empty((T, num_heads, head_dim), dtype=torch.bfloat16, device=q.device)
    elif out.shape != (T, num_heads, head_dim) or out.stride(-1) != 1 or out.stride(1) != head_dim:
        raise ValueError("out must be [tokens, num_heads, head_dim] with contiguous heads")
    args = _lib.PagedAttentionArgs()
    args.q, args.q_row_stride = q.data_ptr(), q.stride(0)
    args.out, args.out_row_stride = out.data_ptr(), out.stride(0)
    args.num_q_rows = T
    code = _lib.KV_BF16
    if k_cache is not None and k_cache.numel():
        code = kv_dtype_code(k_cache)
        if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError("KV pool views must be contiguous")
        if k_cache.dim() != 4 or k_cache.shape[2] != num_kv_heads or k_cache.shape[3] != head_dim:
            raise ValueError("KV pool must be [num_blocks, block_size, num_kv_heads, head_dim]")
        args.k_cache, args.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        args.num_blocks, args.block_size = k_cache.shape[0], k_cache.shape[1]
        if code == _lib.KV_FP8_E4M3FN:
            if k_scale is None or v_scale is None:
                raise ValueError("an E4M3FN pool needs k_scale and v_scale")
            args.k_scale, args.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    args.kv_dtype = code
    decode_cap_len = 0
    if num_decode:
        _int32(decode_lens, "decode_lens")
        _int32(decode_tables, "decode_tables")
        if decode_tables.dim() != 2 or decode_tables.stride(1) != 1:
            raise ValueError("decode_tables must be a row-major [rows, width] int32 tensor")
        if decode_lens.numel() < num_decode or decode_tables.shape[0] < num_decode:
            raise ValueError("decode metadata has fewer rows than num_decode")
        args.num_decode = num_decode
        args.decode_lens = decode_lens.data_ptr()
        args.decode_tables = decode_tables.data_ptr()
        args.decode_table_stride = decode_tables.stride(0)
        args.decode_table_width = decode_tables.shape[1]
        decode_cap_len = decode_tables.shape[1] * args.block_size
    if num_prefill:
        _int32(prefill_cu_q, "cu_seqlens_q")
        _int32(prefill_cu_k, "cu_seqlens_k")
        if prefill_cu_q.numel() < num_prefill + 1 or prefill_cu_k.numel() < num_prefill + 1:
            raise ValueError("cu_seqlens shorter than num_prefill + 1")
        args.num_prefill = num_prefill
        args.prefill_cu_q, args.prefill_cu_k = prefill_cu_q.data_ptr(), prefill_cu_k.data_ptr()
        args.max_q, args.max_k = int(max_q), int(max_k)
        if prefill_tables is not None:
            _int32(prefill_tables, "block_tables")
            if prefill_tables.dim() != 2 or prefill_tables.stride(1) != 1:
                raise ValueError("block_tables must be a row-major [rows, width] int32 tensor")
            args.prefill_tables = prefill_tables.data_ptr()
            args.prefill_table_stride = prefill_tables.stride(0)
            args.prefill_table_width = prefill_tables.shape[1]
        else:
            if k is None or v is None:
                raise ValueError("prefill without block tables needs contiguous k and v")
            for name, t in (("k", k), ("v", v)):
                if t.dtype != torch.bfloat16 or t.stride(-1) != 1 or t.stride(1) != head_dim:
                    raise ValueError(f"{name} must be bf16 [tokens, num_kv_heads, head_dim] rows")
            args.k, args.k_row_stride = k.data_ptr(), k.stride(0)
            args.v, args.v_row_stride = v.data_ptr(), v.stride(0)
            args.num_kv_rows = min(k.shape[0], v.shape[0])
    if store_slot_mapping is not None:
        check_store(new_k, new_v, k_cache, v_cache, store_slot_mapping, k_scale, v_scale)
        if code != _lib.KV_BF16 and num_heads > 8 * num_kv_heads:
            raise ValueError("the E4M3FN KV write in the attention launch needs <= 8 query heads per kv head")
        if new_k.shape[0] != T or new_k.shape[1] != num_kv_heads or new_k.shape[2] != head_dim:
            raise ValueError("new_k/new_v must hold one [num_kv_heads, head_dim] row per query row")
        args.k_cache, args.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        args.num_blocks, args.block_size = k_cache.shape[0], k_cache.shape[1]
        args.store_slot_mapping = store_slot_mapping.data_ptr()
        args.new_k, args.new_k_row_stride = new_k.data_ptr(), new_k.stride(0)
        args.new_v, args.new_v_row_stride = new_v.data_ptr(), new_v.stride(0)
        args.num_new_rows = T
        args.store_scale_floor = float(store_scale_floor)
    args.num_heads, args.num_kv_heads, args.head_dim = num_heads, num_kv_heads, head_dim
    args.softmax_scale = float(softmax_scale)
    args.phases = int(phases)
    if noalloc:
        args.workspace, args.workspace_bytes = None, 0
        _lib.check(_lib.load().slo_paged_attention_noalloc(ctypes.byref(args), _stream(device)),
                   "slo_paged_attention_noalloc")
        return out
    need = _lib.workspace_bytes(num_decode if (phases & _lib.PHASE_DECODE) else 0,
                                decode_cap_len, num_heads, num_kv_heads, head_dim)
    ws = workspace(device, need)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check(_lib.load().slo_paged_attention(ctypes.byref(args), _stream(device)),
               "slo_paged_attention")
    return out


def _paged_attention_fp4(q, k_cache, v_cache, softmax_scale, num_kv_heads, k_scale, v_scale, num_decode, decode_lens,
                         decode_tables, num_prefill, cu_q, cu_k, max_q, max_k, tables, k, v, phases, out, slot_mapping, new_k,
                         new_v, noalloc, scale_floor):
    """``paged_attention`` over a 4-bit pool."""
    index, geometry = _check_query(q, num_kv_heads, k_cache, k_scale, v_cache, v_scale, True, decode_lens, decode_tables, cu_q,
                                   cu_k, tables, k, v, out)
    if noalloc:
        raise ValueError("noalloc launches take bf16 and E4M3FN pools")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    elif out.dtype != torch.bfloat16:
        raise TypeError("out must be bf16")
    elif out.shape != q.shape or out.stride(2) != 1 or out.stride(1) != q.shape[2]:
        raise ValueError("out must be [tokens, num_heads, head_dim] with contiguous heads")
    if slot_mapping is not None:
        store_kvcache(new_k, new_v, k_cache, v_cache, slot_mapping, k_scale, v_scale, scale_floor)
    phases &= _lib.PHASE_ALL
    if num_prefill and tables is None and phases & _lib.PHASE_PREFILL:
        paged_attention(q, None, None, softmax_scale, num_kv_heads=num_kv_heads, num_decode=num_decode, decode_lens=decode_lens,
                        decode_tables=decode_tables, num_prefill=num_prefill, prefill_cu_q=cu_q, prefill_cu_k=cu_k, max_q=max_q,
                        max_k=max_k, k=k, v=v, phases=_lib.PHASE_PREFILL, out=out)
        phases &= ~_lib.PHASE_PREFILL
    rows = _row_args(q.shape[0], num_decode, decode_lens, decode_tables, num_prefill, cu_q, cu_k, max_q, max_k, tables, phases)
    _pool_call("slo_paged_attention_fp4", (), index, q.device, q, out, k_cache, v_cache, k_scale, v_scale, geometry, rows,
               float(softmax_scale), phases)
    return out
