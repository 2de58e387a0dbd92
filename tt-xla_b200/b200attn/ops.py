"""CUDA ops of the attention / KV-cache path, one per `torch.ops.tt.*` op the reference plugin
calls (python_package/tt_torch/custom_ops.py).  Each takes torch CUDA tensors, validates the
layout the reference documents, and calls the C ABI on torch's current stream.

The reference ops are functional (they return a new cache, which the caller copies back,
attention.py:513-515); these update the caches in place, which is what that copy-back amounts
to.
"""
from __future__ import annotations

import ctypes
import functools
import os
import threading
from typing import Optional

import torch

from . import _lib

_workspaces: dict[tuple[int, int], torch.Tensor] = {}
# Scratch that was outgrown stays allocated: a CUDA graph captured earlier still launches into
# it, and its arrival counters must stay zero (memory handed back to the allocator could be
# given to another tensor).
_retired_workspaces: list[torch.Tensor] = []


CACHE_BF16, CACHE_FP8_E4M3, CACHE_INT8 = 0, 1, 2     # enum b200attn_cache_dtype
TICKET_BYTES = 65536                  # B200ATTN_DECODE_TICKET_BYTES


def _cache_dtype(cache: torch.Tensor) -> int:
    if cache.dtype == torch.int8:
        return CACHE_INT8
    return CACHE_FP8_E4M3 if cache.dtype == torch.float8_e4m3fn else CACHE_BF16


def _env_num_splits() -> int:
    """`B200ATTN_NUM_SPLITS=n` pins the split count of every decode call that leaves it to the
    library (for sweeps and for ruling the cost model out while debugging); unset or 0 = the
    model's choice.  Read on every call: changing it between steps is allowed outside graphs."""
    raw = os.environ.get("B200ATTN_NUM_SPLITS", "")
    if not raw:
        return 0
    n = int(raw)
    if not 0 <= n <= 256:
        raise ValueError(f"B200ATTN_NUM_SPLITS must be 0..256, got {raw!r}")
    return n


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _need_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "b200attn ops run on CUDA tensors only (there is no CPU path); got a "
                f"{t.device.type} tensor"
            )


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor,
                 scaled: bool = False) -> tuple[int, int, int, int]:
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(
            "k_cache and v_cache must both be [num_blocks, num_kv_heads, block_size, head_size]; "
            f"got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}"
        )
    if scaled:
        if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (torch.int8, torch.float8_e4m3fn):
            raise ValueError("block-scaled caches must both be int8 or both be float8_e4m3fn")
    elif k_cache.dtype != v_cache.dtype or k_cache.dtype not in (torch.bfloat16,
                                                                 torch.float8_e4m3fn):
        raise ValueError("caches must both be bfloat16 or both be float8_e4m3fn")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    nb, nkv, bs, hd = k_cache.shape
    return nb, nkv, bs, hd


def _token_major(x: torch.Tensor, nheads: int, hd: int, name: str) -> tuple[torch.Tensor, int]:
    """Returns a [tokens, nheads, hd] view whose last two dims are dense, and its row stride."""
    x = x.reshape(-1, nheads, hd) if x.dim() != 3 else x
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16")
    if x.stride(2) != 1 or x.stride(1) != hd:
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else max(x.stride(0), nheads * hd)


def _i32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    return t


# Raw handle of a device's current stream, and the current device, without building Python objects:
# the ops below are a few microseconds long on the GPU.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _device_of(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Index of the CUDA device all tensors are on; raises when they are not."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _need_cuda(first, t)
            raise ValueError(f"all tensors must be on {first.device}, got one on {t.device}")
    if index < 0:
        _need_cuda(first)
    return index


def _check_scales(k_scale, v_scale, k_cache: torch.Tensor) -> bool:
    """True when the caches are block-scaled; the scales are dense fp32 [num_blocks, num_kv_heads]."""
    if k_scale is None and v_scale is None:
        return False
    if k_scale is None or v_scale is None:
        raise ValueError("k_scale and v_scale go together")
    shape = k_cache.shape[:2]
    if k_scale.shape != shape or v_scale.shape != shape or k_scale.dtype != torch.float32 \
            or v_scale.dtype != torch.float32 or not k_scale.is_contiguous() \
            or not v_scale.is_contiguous():
        raise ValueError("k_scale / v_scale must be dense float32 [num_blocks, num_kv_heads]")
    return True


def paged_update_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    update_indices: torch.Tensor,
    page_table: torch.Tensor,
) -> None:
    """Decode-step KV write: `tt.paged_update_cache` for K and V in one launch
    (custom_ops.py:962-1013).  `key`/`value`: [users, nkv, hd] (the reference's
    [1, users, nkv, hd] is accepted too)."""
    _need_cuda(k_cache, v_cache, key, value, update_indices, page_table)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache)
    key, kstride = _token_major(key, nkv, hd, "key")
    value, vstride = _token_major(value, nkv, hd, "value")
    if key.shape != value.shape:
        raise ValueError("key and value must have the same shape")
    if kstride != vstride:
        value = value.contiguous()
        key = key.contiguous()
        kstride = nkv * hd
    users = update_indices.shape[0]
    if key.shape[0] != users or page_table.shape[0] < users:
        raise ValueError("key/value rows, update_indices and page_table rows must agree")
    _i32(update_indices, "update_indices")
    _i32(page_table, "page_table")
    if page_table.stride(1) != 1 or not update_indices.is_contiguous():
        raise ValueError("page_table rows and update_indices must be dense")
    L = _lib.lib()
    _lib.check(
        "b200attn_paged_update_cache_ex",
        L.b200attn_paged_update_cache_ex(
            k_cache.data_ptr(), v_cache.data_ptr(), key.data_ptr(), value.data_ptr(), kstride,
            update_indices.data_ptr(), page_table.data_ptr(), page_table.stride(0),
            page_table.shape[1], users, nkv, hd, bs, nb, _cache_dtype(k_cache), _stream(k_cache),
        ),
    )


def paged_fill_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    fill_page_table: torch.Tensor,
    batch_idx: Optional[torch.Tensor] = None,
) -> None:
    """Prefill / chunk KV write: `tt.paged_fill_cache` for K and V, all users in one launch
    (custom_ops.py:1016-1104).  `key`/`value`: [users, tokens, nkv, hd] token-major (the layout
    the plugin holds before it transposes for the reference op, attention.py:487-488)."""
    _need_cuda(k_cache, v_cache, key, value, fill_page_table, batch_idx)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache)
    if key.dim() != 4 or key.shape != value.shape or key.shape[2] != nkv or key.shape[3] != hd:
        raise ValueError(
            f"key/value must be [users, tokens, {nkv}, {hd}], got {tuple(key.shape)}"
        )
    users, tokens = key.shape[0], key.shape[1]
    if not key.is_contiguous():
        key = key.contiguous()
    if not value.is_contiguous():
        value = value.contiguous()
    _i32(fill_page_table, "fill_page_table")
    if fill_page_table.stride(1) != 1:
        raise ValueError("fill_page_table rows must be dense")
    if batch_idx is not None:
        _i32(batch_idx, "batch_idx")
        if batch_idx.numel() != users or not batch_idx.is_contiguous():
            raise ValueError("batch_idx must hold one dense entry per user")
    L = _lib.lib()
    _lib.check(
        "b200attn_paged_fill_cache_ex",
        L.b200attn_paged_fill_cache_ex(
            k_cache.data_ptr(), v_cache.data_ptr(), key.data_ptr(), value.data_ptr(), nkv * hd,
            fill_page_table.data_ptr(), fill_page_table.stride(0), fill_page_table.shape[1],
            batch_idx.data_ptr() if batch_idx is not None else None,
            users, tokens, nkv, hd, bs, nb, _cache_dtype(k_cache), _stream(k_cache),
        ),
    )


def kv_scatter_slots(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """KV write addressed by vLLM's `slot_mapping` (int64, negative = skip); the live-layout
    counterpart of `write_to_kv_cache` (attention.py:671-716)."""
    _need_cuda(k_cache, v_cache, key, value, slot_mapping)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache)
    key, kstride = _token_major(key, nkv, hd, "key")
    value, vstride = _token_major(value, nkv, hd, "value")
    if kstride != vstride:
        key, value = key.contiguous(), value.contiguous()
        kstride = nkv * hd
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be a dense int64 tensor")
    n = slot_mapping.numel()
    if key.shape[0] < n or value.shape[0] < n:
        raise ValueError("fewer key/value rows than slots")
    L = _lib.lib()
    _lib.check(
        "b200attn_kv_scatter_slots_ex",
        L.b200attn_kv_scatter_slots_ex(
            k_cache.data_ptr(), v_cache.data_ptr(), key.data_ptr(), value.data_ptr(), kstride,
            slot_mapping.data_ptr(), n, nkv, hd, bs, nb, _cache_dtype(k_cache), _stream(k_cache),
        ),
    )


def rope_kv_scatter_slots(
    query: torch.Tensor,
    key: torch.Tensor,
    value: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    rotary_dim: int,
    head_size: int,
    k_cache: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    slot_mapping: Optional[torch.Tensor] = None,
    is_neox_style: bool = True,
) -> None:
    """Rotary embedding of `query` / `key` IN PLACE, computed like the plugin's rotary layer
    (layers/rotary_embedding.py:51-66), fused with the slot-mapping cache write of the rotated
    key and of `value`.  `query` [tokens, nq*hd], `key` / `value` [tokens, nkv*hd] (dense rows,
    any row stride); `positions` int64 [tokens]; `inv_freq` fp32 [rotary_dim/2].  Without
    `slot_mapping` only the rotation is done."""
    _need_cuda(query, key, value, positions, inv_freq, k_cache, v_cache, slot_mapping)
    tokens = positions.numel()
    if query.dim() != 2 or key.dim() != 2 or query.shape[0] != tokens or key.shape[0] != tokens:
        raise ValueError("query / key must be [tokens, heads*head_size] with one row per position")
    if query.dtype != torch.bfloat16 or key.dtype != torch.bfloat16:
        raise ValueError("query / key must be bfloat16")
    if query.stride(1) != 1 or key.stride(1) != 1:
        raise ValueError("query / key rows must be dense")
    nq, nkv = query.shape[1] // head_size, key.shape[1] // head_size
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        raise ValueError("positions must be a dense int64 tensor")
    if inv_freq.dtype != torch.float32 or inv_freq.numel() != rotary_dim // 2 \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be dense float32 [rotary_dim / 2]")
    nb = bs = 0
    if slot_mapping is not None:
        nb, nkv_c, bs, hd_c = _check_cache(k_cache, v_cache)
        if nkv_c != nkv or hd_c != head_size:
            raise ValueError("cache geometry differs from key geometry")
        if value is None or value.shape != key.shape or value.stride(1) != 1:
            raise ValueError("value must match key")
        if slot_mapping.dtype != torch.int64 or slot_mapping.numel() < tokens:
            raise ValueError("slot_mapping must be int64 with one entry per token")
    L = _lib.lib()
    _lib.check(
        "b200attn_rope_kv_scatter_slots",
        L.b200attn_rope_kv_scatter_slots(
            query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0),
            value.data_ptr() if value is not None else None,
            value.stride(0) if value is not None else 0,
            positions.data_ptr(), inv_freq.data_ptr(), rotary_dim, 1 if is_neox_style else 0,
            k_cache.data_ptr() if slot_mapping is not None else None,
            v_cache.data_ptr() if slot_mapping is not None else None,
            slot_mapping.data_ptr() if slot_mapping is not None else None,
            tokens, nq, nkv, head_size, bs, nb, _stream(query),
        ),
    )


def _rows_meet(a: tuple, b: tuple, tokens: int) -> bool:
    """Whether two sets of `tokens` rows, each (pointer, row stride, row width) in bytes, share
    memory.  Exact for equal strides (columns of one buffer), else by the memory between their
    first and last byte."""
    (a0, a_step, a_width), (b0, b_step, b_width) = a, b
    if b0 >= a0 + (tokens - 1) * a_step + a_width or a0 >= b0 + (tokens - 1) * b_step + b_width:
        return False
    if a_step == b_step and a_step > 0:
        gap = (b0 - a0) % a_step
        return gap < a_width or a_step - gap < b_width
    return True


def rows_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the dense rows of two 2-D tensors with as many rows share memory (as exact as
    _rows_meet)."""
    spans = [(t.data_ptr(), t.stride(0) * t.element_size(), t.shape[1] * t.element_size())
             for t in (a, b)]
    return a.shape[0] > 0 and _rows_meet(*spans, a.shape[0])


def _check_outputs(tokens: int, oq: tuple, ok: tuple, q: tuple, k: tuple, v: tuple) -> None:
    """Each output is its input or shares no memory with it, and shares none with the other input,
    with v (read when its pointer is not 0) and with the other output: the kernel stores a token's
    rows while it still reads others of them.  All as (pointer, row stride, row width) in bytes."""
    # the usual case first: outputs on either side of everything else
    last = tokens - 1
    lo = min(q[0], k[0], v[0] or q[0])
    hi = max(q[0] + last * q[1] + q[2], k[0] + last * k[1] + k[2], v[0] + last * v[1] + v[2])
    oq_end, ok_end = oq[0] + last * oq[1] + oq[2], ok[0] + last * ok[1] + ok[2]
    if (oq[0] >= hi or oq_end <= lo) and (ok[0] >= hi or ok_end <= lo) and \
            (oq[0] >= ok_end or ok[0] >= oq_end):
        return
    for out, own, other in ((oq, q, k), (ok, k, q)):
        if _rows_meet(out, other, tokens) or (v[0] and _rows_meet(out, v, tokens)) \
                or (out != own and _rows_meet(out, own, tokens)):
            raise ValueError("an output must be its input or overlap none of the inputs")
    if _rows_meet(oq, ok, tokens):
        raise ValueError("the outputs must not overlap")


def qk_norm_rope_kv_scatter_slots(
    query: torch.Tensor,
    key: torch.Tensor,
    value: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    rotary_dim: int,
    head_size: int,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    eps: float = 1e-6,
    k_cache: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    slot_mapping: Optional[torch.Tensor] = None,
    is_neox_style: bool = True,
    out_query: Optional[torch.Tensor] = None,
    out_key: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head (`q_weight` / `k_weight` [head_size], bf16 or fp32,
    shared by the heads), then the rotary embedding, then, with `slot_mapping`, the cache write of
    the rotated key and of `value`: `rope_kv_scatter_slots` with the per-head norms in front, in one
    pass.  Computed in fp32 (angles in fp64) and rounded to bf16 once.  `query` [tokens, nq*hd],
    `key` / `value` [tokens, nkv*hd], dense rows of any row stride; results go to `out_query` /
    `out_key` of the same shapes, or in place when these are not given.  An output either is its
    input or does not overlap it; it overlaps no other input (nor `value`, when that is written to
    the cache) and not the other output.  Pairs are (i, i + rotary_dim/2) for `is_neox_style`,
    (2i, 2i + 1) otherwise.  Caches: bf16 or unscaled e4m3 (`paged_write` fills block-scaled
    ones).  Returns (out_query, out_key)."""
    oq = query if out_query is None else out_query
    ok = key if out_key is None else out_key
    index = _device_of(query, key, positions, inv_freq, q_weight, k_weight, out_query, out_key,
                       value, slot_mapping, k_cache, v_cache)
    if _current_device() != index:       # the library works on the current device
        with torch.cuda.device(index):
            return qk_norm_rope_kv_scatter_slots(
                query, key, value, positions, inv_freq, rotary_dim, head_size, q_weight, k_weight,
                eps, k_cache, v_cache, slot_mapping, is_neox_style, out_query, out_key)
    tokens = positions.numel()
    if query.dim() != 2 or key.dim() != 2 or query.shape[0] != tokens or key.shape[0] != tokens:
        raise ValueError("query / key must be [tokens, heads*head_size] with one row per position")
    q_width, k_width = query.shape[1], key.shape[1]
    if q_width % head_size or k_width % head_size:
        raise ValueError("query / key rows must hold whole heads")
    bf16 = torch.bfloat16
    if query.dtype != bf16 or key.dtype != bf16 or query.stride(1) != 1 or key.stride(1) != 1:
        raise ValueError("query / key must be bfloat16 with dense rows")
    q_stride, k_stride = (query.stride(0), key.stride(0)) if tokens > 1 else (q_width, k_width)
    oq_stride, ok_stride = q_stride, k_stride
    if oq is not query or ok is not key:
        if oq.shape != query.shape or ok.shape != key.shape:
            raise ValueError("out_query / out_key must have query's / key's shape")
        if oq.dtype != bf16 or ok.dtype != bf16 or oq.stride(1) != 1 or ok.stride(1) != 1:
            raise ValueError("out_query / out_key must be bfloat16 with dense rows")
        if tokens > 1:
            oq_stride, ok_stride = oq.stride(0), ok.stride(0)
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        raise ValueError("positions must be a dense int64 tensor")
    if inv_freq.dtype != torch.float32 or inv_freq.numel() != rotary_dim // 2 \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be dense float32 [rotary_dim / 2]")
    w_dtype = q_weight.dtype
    if w_dtype != k_weight.dtype or w_dtype not in (bf16, torch.float32):
        raise ValueError("q_weight / k_weight must both be bfloat16 or both be float32")
    if q_weight.numel() != head_size or k_weight.numel() != head_size \
            or not q_weight.is_contiguous() or not k_weight.is_contiguous():
        raise ValueError("q_weight / k_weight must be dense [head_size]")
    nkv = k_width // head_size
    nb = bs = v_stride = v_ptr = kc_ptr = vc_ptr = slot_ptr = kind = 0
    if slot_mapping is not None:
        if k_cache is None or v_cache is None or value is None:
            raise ValueError("slot_mapping needs k_cache, v_cache and value")
        nb, nkv_c, bs, hd_c = _check_cache(k_cache, v_cache)
        if nkv_c != nkv or hd_c != head_size:
            raise ValueError("cache geometry differs from key geometry")
        if value.shape != key.shape or value.dtype != bf16 or value.stride(1) != 1:
            raise ValueError("value must match key")
        if slot_mapping.dtype != torch.int64 or slot_mapping.numel() < tokens \
                or not slot_mapping.is_contiguous():
            raise ValueError("slot_mapping must be dense int64 with one entry per token")
        v_stride = value.stride(0) if tokens > 1 else k_width
        v_ptr, kc_ptr, vc_ptr = value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
        slot_ptr, kind = slot_mapping.data_ptr(), _cache_dtype(k_cache)
    if tokens == 0:
        return oq, ok
    oq_ptr, ok_ptr, q_ptr, k_ptr = oq.data_ptr(), ok.data_ptr(), query.data_ptr(), key.data_ptr()
    _check_outputs(tokens, (oq_ptr, 2 * oq_stride, 2 * q_width),
                   (ok_ptr, 2 * ok_stride, 2 * k_width), (q_ptr, 2 * q_stride, 2 * q_width),
                   (k_ptr, 2 * k_stride, 2 * k_width), (v_ptr, 2 * v_stride, 2 * k_width))
    status = _lib.lib().b200attn_qk_norm_rope_kv_scatter_slots(
        oq_ptr, oq_stride, ok_ptr, ok_stride, q_ptr, q_stride, k_ptr, k_stride,
        v_ptr, v_stride, q_weight.data_ptr(), k_weight.data_ptr(),
        1 if w_dtype == torch.float32 else 0, eps, positions.data_ptr(), inv_freq.data_ptr(),
        rotary_dim, 1 if is_neox_style else 0, kc_ptr, vc_ptr, kind, slot_ptr, tokens,
        q_width // head_size, nkv, head_size, bs, nb, _raw_stream(index))
    if status:
        _lib.check("b200attn_qk_norm_rope_kv_scatter_slots", status)
    return oq, ok


def _rows_3d(x: torch.Tensor, nheads: int, hd: int, name: str) -> tuple[torch.Tensor, int]:
    """[tokens, nheads, hd] view of bf16 rows with dense heads, and the row stride."""
    if x.dim() == 2 and x.shape[1] == nheads * hd:
        x = x.unflatten(1, (nheads, hd))
    if x.dim() != 3 or tuple(x.shape[1:]) != (nheads, hd):
        raise ValueError(f"{name} must be [tokens, {nheads}, {hd}], got {tuple(x.shape)}")
    return _token_major(x, nheads, hd, name)


def paged_write(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    page_table: torch.Tensor,
    q_start: torch.Tensor,
    cu_q: Optional[torch.Tensor] = None,
    q_len: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    k_bounds: Optional[torch.Tensor] = None,
) -> None:
    """Varlen KV write that keeps per-page values.  Rows `cu_q[s]:cu_q[s+1]` of `key` / `value`
    ([tokens, nkv, hd] bf16) go to positions `q_start[s]`, `q_start[s] + 1`, ... of sequence s
    through `page_table[s]`; without `cu_q` every sequence has one token.  `q_len` limits how many of
    a sequence's rows are written (padded batches); a negative `q_start` skips the sequence.

    Caches: int8 or float8_e4m3fn with `k_scale` / `v_scale` (fp32 [num_blocks, num_kv_heads], an
    element reads as code * scale), or bf16 without scales (`k_bounds` is then what the call is
    for).  A page whose first row is written starts afresh; one that goes on grows its scale by a
    power of two when a new row needs it and re-rounds the rows that stay: those before the first
    new one (what lies behind the new rows counts as free).  A NaN or infinity makes
    the scale NaN, and with it everything read through the page.  `k_bounds` (bf16 [num_blocks,
    num_kv_heads, 2, head_size]) keeps the least and greatest key of each channel for
    `select_pages`.  The sequences of one call must write to different pages."""
    index = _device_of(k_cache, v_cache, key, value, page_table, q_start, cu_q, q_len, k_scale,
                       v_scale, k_bounds)
    if _current_device() != index:       # the library works on the current device
        with torch.cuda.device(index):
            return paged_write(k_cache, v_cache, key, value, page_table, q_start, cu_q, q_len,
                               k_scale, v_scale, k_bounds)
    scaled = _check_scales(k_scale, v_scale, k_cache)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache, scaled)
    if not scaled:
        if k_cache.dtype != torch.bfloat16:
            raise ValueError("an 8-bit cache needs k_scale and v_scale here (kv_scatter_slots "
                             "writes unscaled e4m3)")
        if k_bounds is None:
            raise ValueError("a bf16 cache without k_bounds is kv_scatter_slots's")
    if k_bounds is not None and (k_bounds.dtype != torch.bfloat16 or not k_bounds.is_contiguous()
                                 or k_bounds.shape != (nb, nkv, 2, hd)):
        raise ValueError("k_bounds must be dense bfloat16 [num_blocks, num_kv_heads, 2, head_size]")
    key, kstride = _rows_3d(key, nkv, hd, "key")
    value, vstride = _rows_3d(value, nkv, hd, "value")
    rows = key.shape[0]
    if value.shape[0] != rows:
        raise ValueError("key and value must have the same shape")
    i32 = torch.int32
    seqs = q_start.numel()
    if page_table.dtype != i32 or page_table.dim() != 2 or page_table.shape[0] < seqs \
            or page_table.stride(1) != 1:
        raise ValueError("page_table must be int32 with a dense row per sequence")
    if q_start.dtype != i32 or not q_start.is_contiguous():
        raise ValueError("q_start must be int32 with a dense entry per sequence")
    if cu_q is None:
        if rows != seqs:
            raise ValueError("without cu_q, key / value must hold one row per sequence")
    elif cu_q.dtype != i32 or cu_q.numel() != seqs + 1 or not cu_q.is_contiguous():
        raise ValueError("cu_q must be int32 with num_seqs + 1 dense entries")
    if q_len is not None and (q_len.dtype != i32 or q_len.numel() != seqs
                              or not q_len.is_contiguous()):
        raise ValueError("q_len must be int32 with a dense entry per sequence")
    if seqs == 0 or rows == 0:
        return
    status = _lib.lib().b200attn_paged_write(
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr() if scaled else 0,
        v_scale.data_ptr() if scaled else 0, 0 if k_bounds is None else k_bounds.data_ptr(),
        _cache_dtype(k_cache), key.data_ptr(), kstride, value.data_ptr(), vstride,
        page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
        0 if cu_q is None else cu_q.data_ptr(), 0 if q_len is None else q_len.data_ptr(),
        q_start.data_ptr(), seqs, rows, nkv, hd, bs, nb, _raw_stream(index))
    if status:
        _lib.check("b200attn_paged_write", status)


def decode_auto_splits(users: int, nkv: int, hd: int, max_context_len: int) -> int:
    return _lib.lib().b200attn_decode_auto_splits(users, nkv, hd, max_context_len)


def decode_workspace_bytes(users: int, nq: int, hd: int, splits: int) -> int:
    return _lib.lib().b200attn_decode_workspace_bytes(users, nq, hd, splits)


def _workspace(device: torch.device, nbytes: int) -> Optional[torch.Tensor]:
    """Split-KV scratch, cached per (device, stream) and grown on demand.  torch owns the
    memory; the C library never allocates.  Allocated zeroed: the arrival counters at its start
    have to be zero on first use (every call leaves them zero)."""
    if nbytes == 0:
        return None
    key = (device.index or 0, torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _retired_workspaces.append(ws)
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


_capture_workspaces: dict[tuple[int, int], tuple[int, torch.Tensor]] = {}


def _scratch(index: int, stream: int, nbytes: int) -> Optional[torch.Tensor]:
    """Scratch of the block-scaled and page-list ops on the (current) device `index`.  Eager calls
    take the stream's workspace.  Calls under stream capture take one that belongs to the graph
    being captured (from its memory pool, its counters zeroed by a node of the graph), so that
    graphs captured on the same stream may be replayed side by side on others."""
    if nbytes == 0:
        return None
    key = (index, stream)
    if not torch.cuda.is_current_stream_capturing():
        ws = _workspaces.get(key)
        return ws if ws is not None and ws.numel() >= nbytes else \
            _workspace(torch.device("cuda", index), nbytes)
    capture = ctypes.c_uint64(0)
    _lib.check("b200attn_capture_id",
               _lib.lib().b200attn_capture_id(ctypes.byref(capture), stream))
    have = _capture_workspaces.get(key)
    if have is None or have[0] != capture.value or have[1].numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=torch.device("cuda", index))
        ws[:TICKET_BYTES].zero_()
        have = (capture.value, ws)
        _capture_workspaces[key] = have
    return have[1]


# Sizes and split counts are functions of whole numbers, and where the SM count is among them of the
# device (which is the current one when they are asked for).
@functools.lru_cache(maxsize=4096)
def _select_bytes(users: int, nkv: int, width: int) -> int:
    return _lib.lib().b200attn_select_pages_workspace_bytes(users, nkv, width)


@functools.lru_cache(maxsize=4096)
def _list_splits(device: int, users: int, nkv: int, hd: int, ctx: int) -> int:
    return _lib.lib().b200attn_decode_auto_splits(users, nkv, hd, ctx)


@functools.lru_cache(maxsize=4096)
def _decode_bytes(users: int, nq: int, hd: int, splits: int) -> int:
    return _lib.lib().b200attn_decode_workspace_bytes(users, nq, hd, splits)


@functools.lru_cache(maxsize=4096)
def _scaled_bytes(device: int, users: int, nq: int, nkv: int, hd: int, splits: int) -> int:
    return _lib.lib().b200attn_decode_scaled_workspace_bytes(users, nq, nkv, hd, splits)


def select_pages(
    query: torch.Tensor,
    k_bounds: torch.Tensor,
    page_table: torch.Tensor,
    cur_pos: torch.Tensor,
    block_size: int,
    num_pages: int,
    keep_first: int = 1,
    keep_last: int = 1,
    max_context_len: int = 0,
    workspace: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Chooses, for every user and KV head, the `num_pages` pages of the context a block-sparse
    decode attends to: all of them when there are no more, else the first `keep_first`, the last
    `keep_last` (>= 1) and those whose key bounds allow the largest logit of any of the head's
    queries (equal scores: the lower page).  `query` [users, nq, hd]; `k_bounds` as `paged_write`
    keeps them; `page_table` [users, width] and `cur_pos` [users] as for `paged_decode`.
    Returns (table [users, nkv, num_pages], pos [users, nkv]): hand them to `paged_decode` as
    `page_table` and `cur_pos`.  A position behind the table is reported (diagnostics word 2) and
    gives the choice at the table's last key.  `max_context_len` only shapes the launch."""
    index = _device_of(query, k_bounds, page_table, cur_pos, workspace)
    if _current_device() != index:       # the library works on the current device
        with torch.cuda.device(index):
            return select_pages(query, k_bounds, page_table, cur_pos, block_size, num_pages,
                                keep_first, keep_last, max_context_len, workspace)
    if k_bounds.dim() != 4 or k_bounds.shape[2] != 2 or k_bounds.dtype != torch.bfloat16 \
            or not k_bounds.is_contiguous():
        raise ValueError("k_bounds must be dense bfloat16 [num_blocks, num_kv_heads, 2, head_size]")
    nb, nkv, _, hd = k_bounds.shape
    if query.dim() == 4 and query.shape[0] == 1:
        query = query[0]
    if query.dim() != 3 or query.shape[2] != hd:
        raise ValueError(f"query must be [users, nq, {hd}], got {tuple(query.shape)}")
    users, nq, _ = query.shape
    if nq % nkv != 0:
        raise ValueError(f"num_q_heads {nq} is not a multiple of num_kv_heads {nkv}")
    q, qstride = _token_major(query, nq, hd, "query")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] < users \
            or page_table.stride(1) != 1 or page_table.shape[1] == 0:
        raise ValueError("page_table must be int32 with a dense row per user")
    if cur_pos.dtype != torch.int32 or not cur_pos.is_contiguous() or cur_pos.numel() != users:
        raise ValueError("cur_pos must be int32 with a dense entry per user")
    if keep_first < 0 or keep_last < 1 or keep_first + keep_last > num_pages:
        raise ValueError("keep_first >= 0 and keep_last >= 1 must fit into num_pages")
    table = cur_pos.new_empty((users, nkv, num_pages))
    pos = cur_pos.new_empty((users, nkv))
    if users == 0:
        return table, pos
    width = page_table.shape[1]
    stream = _raw_stream(index)
    ws = workspace
    if ws is None:
        ws = _scratch(index, stream, _select_bytes(users, nkv, width))
    status = _lib.lib().b200attn_select_pages(
        table.data_ptr(), pos.data_ptr(), q.data_ptr(), qstride, k_bounds.data_ptr(),
        page_table.data_ptr(), page_table.stride(0), width, cur_pos.data_ptr(), users, nq, nkv,
        hd, block_size, nb, num_pages, keep_first, keep_last, max_context_len, ws.data_ptr(),
        ws.numel() * ws.element_size(), stream)
    if status:
        _lib.check("b200attn_select_pages", status)
    return table, pos


def _decode_blocks(query, k_cache, v_cache, page_table, cur_pos, scale, out, num_splits,
                   max_context_len, workspace, sliding_window, sinks, k_scale, v_scale):
    """paged_decode over block-scaled caches and / or a page list per KV head."""
    index = _device_of(query, k_cache, v_cache, page_table, cur_pos, k_scale, v_scale, out, sinks,
                       workspace)
    if _current_device() != index:       # the library works on the current device
        with torch.cuda.device(index):
            return _decode_blocks(query, k_cache, v_cache, page_table, cur_pos, scale, out,
                                  num_splits, max_context_len, workspace, sliding_window, sinks,
                                  k_scale, v_scale)
    scaled = _check_scales(k_scale, v_scale, k_cache)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache, scaled)
    shape = query.shape
    if query.dim() == 4 and shape[0] == 1:
        query = query[0]
    if query.dim() != 3 or query.shape[2] != hd:
        raise ValueError(f"query must be [users, nq, {hd}], got {tuple(shape)}")
    users, nq, _ = query.shape
    if nq % nkv != 0:
        raise ValueError(f"num_q_heads {nq} is not a multiple of num_kv_heads {nkv}")
    q, qstride = _token_major(query, nq, hd, "query")
    if out is None:
        out_t = q.new_empty((users, nq, hd))
    else:
        out_t = out.reshape(users, nq, hd) if out.dim() != 3 else out
        if out_t.shape != q.shape or out_t.dtype != torch.bfloat16 or out_t.stride(2) != 1 \
                or out_t.stride(1) != hd:
            raise ValueError("out must be a dense-row bfloat16 tensor of query's shape")
        if out_t.data_ptr() != out.data_ptr():
            raise ValueError("out must be viewable as [users, nq, hd] without a copy")
    ostride = out_t.stride(0) if users > 1 else max(out_t.stride(0), nq * hd)
    if page_table.dtype != torch.int32 or cur_pos.dtype != torch.int32:
        raise ValueError("page_table and cur_pos must be int32")
    if page_table.stride(-1) != 1 or not cur_pos.is_contiguous():
        raise ValueError("page_table rows and cur_pos must be dense")
    width = page_table.shape[-1]
    head_stride = 0
    if page_table.dim() == 3:
        if page_table.shape[0] != users or page_table.shape[1] != nkv:
            raise ValueError("a page list per KV head must be [users, num_kv_heads, pages]")
        if cur_pos.shape != (users, nkv):
            raise ValueError("with a page list per KV head cur_pos must be [users, num_kv_heads]")
        if sliding_window > 0:
            raise ValueError("a list of chosen pages has no sliding window")
        head_stride = page_table.stride(1) if nkv > 1 else max(page_table.stride(1), width)
        if head_stride < width:
            raise ValueError("the page lists of the KV heads must not overlap")
        max_context_len = min(max_context_len, width * bs)
    elif page_table.dim() != 2 or page_table.shape[0] < users or cur_pos.numel() != users:
        raise ValueError("page_table needs a row, and cur_pos an entry, per user")
    if sinks is not None and (sinks.dtype != torch.float32 or sinks.numel() != nq
                              or not sinks.is_contiguous()):
        raise ValueError("sinks must be a dense float32 tensor with one entry per q head")
    if users == 0:
        return out if out is not None else out_t.reshape(shape)
    stream = _raw_stream(index)
    if num_splits == 0:
        num_splits = _env_num_splits()
    ws = workspace
    if scaled:
        if ws is None:
            ws = _scratch(index, stream, _scaled_bytes(index, users, nq, nkv, hd, num_splits))
    else:
        if num_splits == 0:
            num_splits = _list_splits(index, users, nkv, hd,
                                      max_context_len if max_context_len > 0 else width * bs)
        if ws is None and num_splits > 1:
            ws = _scratch(index, stream, _decode_bytes(users, nq, hd, num_splits))
    status = _lib.lib().b200attn_paged_decode_blocks(
        out_t.data_ptr(), ostride, q.data_ptr(), qstride, k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr() if scaled else 0, v_scale.data_ptr() if scaled else 0,
        _cache_dtype(k_cache), page_table.data_ptr(), page_table.stride(0), head_stride, width,
        cur_pos.data_ptr(), users, nq, nkv, hd, bs, nb, hd ** -0.5 if scale is None else scale,
        sliding_window, sinks.data_ptr() if sinks is not None else 0, max_context_len, num_splits,
        ws.data_ptr() if ws is not None else 0,
        ws.numel() * ws.element_size() if ws is not None else 0, stream)
    if status:
        _lib.check("b200attn_paged_decode_blocks", status)
    return out if out is not None else out_t.reshape(shape)


def paged_decode(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cur_pos: torch.Tensor,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    num_splits: int = 0,
    max_context_len: int = 0,
    workspace: Optional[torch.Tensor] = None,
    sliding_window: int = 0,
    sinks: Optional[torch.Tensor] = None,
    new_key: Optional[torch.Tensor] = None,
    new_value: Optional[torch.Tensor] = None,
    wrap_negative_positions: bool = True,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Paged GQA decode attention: `tt.paged_scaled_dot_product_attention_decode` with
    is_causal=True and cur_pos_tensor (custom_ops.py:1198-1331).  `query`: [users, nq, hd]
    (or the reference's [1, users, nq, hd]); returns / fills `out` of the same shape.
    `sliding_window` > 0 limits each user to its last `sliding_window` keys; `sinks` (fp32
    [nq]) adds one denominator-only softmax column per head (the op's `sliding_window_size` /
    `attention_sink` arguments, which the reference CPU branch ignores).
    With `new_key` / `new_value` ([users, nkv, hd] bf16) the same launch first writes those rows
    into the caches at `cur_pos`, i.e. it is `paged_update_cache` + decode in one kernel;
    `wrap_negative_positions=False` skips rows with a negative position instead of wrapping them
    the way the reference's CPU indexing does.
    `k_scale` / `v_scale` (fp32 [num_blocks, num_kv_heads]): int8 or e4m3 caches with a scale per
    page and KV head, as `paged_write` fills them.  A `page_table` [users, nkv, pages] with a
    `cur_pos` [users, nkv] gives every KV head its own list of pages, `cur_pos` counting within the
    list: what `select_pages` returns (no `sliding_window` then).  Neither form takes `new_key`."""
    if k_scale is not None or v_scale is not None or page_table.dim() == 3:
        if new_key is not None or new_value is not None:
            raise ValueError("new_key / new_value go with unscaled caches and one page list per "
                             "user; use paged_write first")
        return _decode_blocks(query, k_cache, v_cache, page_table, cur_pos, scale, out, num_splits,
                              max_context_len, workspace, sliding_window, sinks, k_scale, v_scale)
    _need_cuda(query, k_cache, v_cache, page_table, cur_pos, out, new_key, new_value)
    nb, nkv, bs, hd = _check_cache(k_cache, v_cache)
    orig_shape = query.shape
    if query.dim() == 4:
        if query.shape[0] != 1:
            raise ValueError("4-D query must be [1, users, nq, hd]")
        query = query[0]
    if query.dim() != 3 or query.shape[2] != hd:
        raise ValueError(f"query must be [users, nq, {hd}], got {tuple(orig_shape)}")
    users, nq = query.shape[0], query.shape[1]
    if nq % nkv != 0:
        raise ValueError(f"num_q_heads {nq} is not a multiple of num_kv_heads {nkv}")
    q, qstride = _token_major(query, nq, hd, "query")
    if out is None:
        out_t = torch.empty((users, nq, hd), dtype=torch.bfloat16, device=query.device)
    else:
        out_t = out.reshape(users, nq, hd) if out.dim() != 3 else out
        if out_t.dtype != torch.bfloat16 or out_t.stride(2) != 1 or out_t.stride(1) != hd:
            raise ValueError("out must be a dense-row bfloat16 tensor")
        if out_t.data_ptr() != out.data_ptr():
            raise ValueError("out must be viewable as [users, nq, hd] without a copy")
    ostride = out_t.stride(0) if users > 1 else max(out_t.stride(0), nq * hd)
    _i32(page_table, "page_table")
    _i32(cur_pos, "cur_pos")
    if page_table.stride(1) != 1 or not cur_pos.is_contiguous() or cur_pos.numel() != users:
        raise ValueError("page_table rows must be dense and cur_pos must hold one entry per user")
    if scale is None:
        scale = hd ** -0.5
    L = _lib.lib()
    if sinks is not None:
        _need_cuda(sinks)
        if sinks.dtype != torch.float32 or sinks.numel() != nq or not sinks.is_contiguous():
            raise ValueError("sinks must be a dense float32 tensor with one entry per q head")
    if num_splits == 0:
        num_splits = _env_num_splits()
    if num_splits == 0:
        ctx = max_context_len if max_context_len > 0 else page_table.shape[1] * bs
        if sliding_window > 0:
            ctx = min(ctx, sliding_window + 64)
        num_splits = L.b200attn_decode_auto_splits(users, nkv, hd, ctx)
    need = L.b200attn_decode_workspace_bytes(users, nq, hd, num_splits)
    ws = workspace if workspace is not None else _workspace(query.device, need)
    kn = vn = None
    nstride = 0
    if (new_key is None) != (new_value is None):
        raise ValueError("new_key and new_value go together")
    if new_key is not None:
        kn, nstride = _token_major(new_key, nkv, hd, "new_key")
        vn, vstride = _token_major(new_value, nkv, hd, "new_value")
        if kn.shape[0] != users or vn.shape[0] != users:
            raise ValueError("new_key / new_value must hold one row per user")
        if vstride != nstride:
            kn, vn, nstride = kn.contiguous(), vn.contiguous(), nkv * hd
    _lib.check(
        "b200attn_paged_decode_step",
        L.b200attn_paged_decode_step(
            out_t.data_ptr(), ostride, q.data_ptr(), qstride, k_cache.data_ptr(),
            v_cache.data_ptr(), kn.data_ptr() if kn is not None else None,
            vn.data_ptr() if vn is not None else None, nstride,
            1 if wrap_negative_positions else 0,
            page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
            cur_pos.data_ptr(), users, nq, nkv, hd, bs, nb, float(scale), int(sliding_window),
            sinks.data_ptr() if sinks is not None else None, _cache_dtype(k_cache), max_context_len,
            num_splits, ws.data_ptr() if ws is not None else None,
            ws.numel() * ws.element_size() if ws is not None else 0, _stream(query),
        ),
    )
    if out is not None:
        return out
    return out_t.reshape(orig_shape)


def prefill(
    query: torch.Tensor,
    k_src: torch.Tensor,
    v_src: torch.Tensor,
    cu_q_host: torch.Tensor,
    scale: Optional[float] = None,
    page_table: Optional[torch.Tensor] = None,
    q_start: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    cu_q: Optional[torch.Tensor] = None,
    sliding_window: int = 0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    max_context_len: int = 0,
) -> torch.Tensor:
    """Causal varlen prefill (`tt.scaled_dot_product_attention`, custom_ops.py:635-742) when
    `page_table` is None and `k_src`/`v_src` are the fresh [tokens, nkv, hd] K/V of the same
    tokens; chunked prefill over the paged cache
    (`tt.chunked_scaled_dot_product_attention`, custom_ops.py:1334-1443) when `page_table` is
    given and `k_src`/`v_src` are the caches.  `query`: [tokens, nq, hd] with sequence s owning
    rows cu_q[s]:cu_q[s+1]; `q_start[s]` is the absolute position of its first row.
    `k_scale` / `v_scale`: paged int8 or e4m3 caches with a scale per page and KV head
    (`paged_write`).  For these the pages that the batch reads are widened into memory of the call,
    as many columns of the page table as `max_context_len` takes (0: all of them).  It must not be
    less than any sequence's q_start + rows: a longer context is reported (diagnostics word 2).
    Under stream capture all columns are taken, since a replay may have longer contexts."""
    if k_scale is None:                      # else _device_of looks at all of them below
        _need_cuda(query, k_src, v_src, page_table, q_start, out, cu_q)
    if cu_q_host.is_cuda or cu_q_host.dtype != torch.int32 or not cu_q_host.is_contiguous():
        raise ValueError("cu_q_host must be a dense int32 CPU tensor")
    num_seqs = cu_q_host.numel() - 1
    if query.dim() != 3:
        raise ValueError(f"query must be [tokens, nq, hd], got {tuple(query.shape)}")
    total_q, nq, hd = query.shape
    q, qstride = _token_major(query, nq, hd, "query")
    paged = page_table is not None
    scaled = False
    if not paged and (k_scale is not None or v_scale is not None):
        raise ValueError("k_scale / v_scale go with a paged cache")
    if paged and k_scale is not None:
        index = _device_of(query, k_src, v_src, page_table, q_start, cu_q, out, k_scale, v_scale)
        if _current_device() != index:       # the library works on the current device
            with torch.cuda.device(index):
                return prefill(query, k_src, v_src, cu_q_host, scale, page_table, q_start, out,
                               cu_q, sliding_window, k_scale, v_scale, max_context_len)
    if paged:
        scaled = _check_scales(k_scale, v_scale, k_src)
        nb, nkv, bs, _hd = _check_cache(k_src, v_src, scaled)
        if _hd != hd:
            raise ValueError("cache head_size differs from query head_size")
        _i32(page_table, "page_table")
        if page_table.stride(1) != 1 or page_table.shape[0] < num_seqs:
            raise ValueError("page_table must have one dense row per sequence")
        kstride = 0
        k, v = k_src, v_src
    else:
        if q_start is not None:
            raise ValueError("q_start needs the paged form (the prefix lives in the cache)")
        if k_src.dim() != 3 or k_src.shape != v_src.shape or k_src.shape[2] != hd:
            raise ValueError("fresh k_src/v_src must be [tokens, nkv, hd]")
        if k_src.shape[0] != total_q:
            raise ValueError("fresh K/V must cover the same tokens as the query")
        nkv = k_src.shape[1]
        k, kstride = _token_major(k_src, nkv, hd, "k_src")
        v, vstride = _token_major(v_src, nkv, hd, "v_src")
        if kstride != vstride:
            k, v = k.contiguous(), v.contiguous()
            kstride = nkv * hd
        nb, bs = 0, 64
    if nq % nkv != 0:
        raise ValueError(f"num_q_heads {nq} is not a multiple of num_kv_heads {nkv}")
    if q_start is not None:
        _i32(q_start, "q_start")
        if q_start.numel() != num_seqs or not q_start.is_contiguous():
            raise ValueError("q_start must hold one dense entry per sequence")
    if cu_q is None:
        cu_q = cu_q_host.to(query.device, non_blocking=True)
    _i32(cu_q, "cu_q")
    if out is None:
        out_t = torch.empty((total_q, nq, hd), dtype=torch.bfloat16, device=query.device)
    else:
        out_t = out.reshape(total_q, nq, hd) if out.dim() != 3 else out
        if out_t.dtype != torch.bfloat16 or out_t.stride(2) != 1 or out_t.stride(1) != hd:
            raise ValueError("out must be a dense-row bfloat16 tensor")
        if out_t.data_ptr() != out.data_ptr():
            raise ValueError("out must be viewable as [tokens, nq, hd] without a copy")
    ostride = out_t.stride(0) if total_q > 1 else max(out_t.stride(0), nq * hd)
    if scale is None:
        scale = hd ** -0.5
    if scaled:
        pool, k_ptr, v_ptr, factors, table, width, nb = _widen_scaled_pages(
            k_src, v_src, k_scale, v_scale, page_table, cu_q, q_start, num_seqs, max_context_len)
        status = _lib.lib().b200attn_prefill_scaled(
            out_t.data_ptr(), ostride, q.data_ptr(),
            qstride if total_q > 1 else max(qstride, nq * hd), k_ptr, v_ptr, factors,
            table.data_ptr(), width, width, cu_q.data_ptr(), cu_q_host.data_ptr(),
            q_start.data_ptr() if q_start is not None else 0, num_seqs, total_q, nq, nkv, hd, bs, nb,
            scale, sliding_window, _raw_stream(index))
        if status:
            _lib.check("b200attn_prefill_scaled", status)
        return out if out is not None else out_t

    def attend(k, v, page_table, nb):
        _lib.check(
            "b200attn_prefill_ex",
            _lib.lib().b200attn_prefill_ex(
                out_t.data_ptr(), ostride, q.data_ptr(), qstride, k.data_ptr(), v.data_ptr(),
                1 if paged else 0, kstride,
                page_table.data_ptr() if paged else None,
                page_table.stride(0) if paged else 0, page_table.shape[1] if paged else 0,
                cu_q.data_ptr(), cu_q_host.data_ptr(),
                q_start.data_ptr() if q_start is not None else None,
                num_seqs, total_q, nq, nkv, hd, bs, nb, float(scale), int(sliding_window),
                _stream(query),
            ),
        )

    if paged and k_src.dtype == torch.float8_e4m3fn:
        # The tcgen05 kernel takes 16-bit tiles: widen the pages this batch reads into a bf16
        # scratch pool laid out [sequence][page slot] and attend over that through the identity
        # page table.  e4m3 -> bf16 is exact, so the kernel sees the cache's own values.  The pool
        # is shared by the calls on a stream, so no other thread may come between the two launches.
        with _fp8_lock:
            attend(*_widen_fp8_pages(k_src, v_src, page_table, cu_q, q_start, num_seqs))
    else:
        attend(k, v, page_table, nb)
    return out if out is not None else out_t


_fp8_scratch: dict[tuple, tuple] = {}
_fp8_lock = threading.Lock()


def _widen_fp8_pages(k_cache, v_cache, page_table, cu_q, q_start, num_seqs):
    """bf16 copies of the pages `page_table[:num_seqs]` lists for an e4m3 cache pair; returns
    (k_pool, v_pool, identity page table, pool size in pages).  The scratch is cached per
    (device, stream) and grown on demand; torch owns it, and _fp8_lock is held from here to the
    launch that reads it."""
    nb, nkv, bs, hd = k_cache.shape
    width = page_table.shape[1]
    pages = num_seqs * width
    dev = k_cache.device
    key = (dev.index or 0, torch.cuda.current_stream(dev).cuda_stream, nkv, bs, hd)
    have = _fp8_scratch.get(key)
    if have is None or have[0].shape[0] < pages:
        if have is not None:
            _retired_workspaces.extend(have[:2])
        grow = max(pages, 2 * have[0].shape[0] if have is not None else 0)
        have = (torch.empty((grow, nkv, bs, hd), dtype=torch.bfloat16, device=dev),
                torch.empty((grow, nkv, bs, hd), dtype=torch.bfloat16, device=dev), {})
        _fp8_scratch[key] = have
    k_pool, v_pool, tables = have
    ident = tables.get((num_seqs, width))
    if ident is None:
        ident = torch.arange(pages, dtype=torch.int32, device=dev).reshape(num_seqs, width)
        tables[(num_seqs, width)] = ident
    _lib.check(
        "b200attn_dequant_pages_fp8",
        _lib.lib().b200attn_dequant_pages_fp8(
            k_pool.data_ptr(), v_pool.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            page_table.data_ptr(), page_table.stride(0), width, cu_q.data_ptr(),
            q_start.data_ptr() if q_start is not None else None, num_seqs, nkv, hd, bs, nb,
            torch.cuda.current_stream(dev).cuda_stream,
        ),
    )
    return k_pool, v_pool, ident, k_pool.shape[0]


_identity_tables: dict[tuple, torch.Tensor] = {}


def _identity_table(device: torch.device, stream: int, pages: int, capturing: bool) -> torch.Tensor:
    """int32 0, 1, 2, ... for `pages` or more pages on the current device: one tensor per stream that
    grows on demand; under stream capture one of the graph's own."""
    if capturing:
        return torch.arange(pages, dtype=torch.int32, device=device)
    have = _identity_tables.get((device.index, stream))
    if have is None or have.numel() < pages:
        have = torch.arange(max(4096, 1 << (pages - 1).bit_length()), dtype=torch.int32, device=device)
        _identity_tables[(device.index, stream)] = have
    return have


def _widen_scaled_pages(k_cache, v_cache, k_scale, v_scale, page_table, cu_q, q_start, num_seqs,
                        max_context_len=0):
    """bf16 pages, laid out as _widen_fp8_pages does, of a block-scaled cache pair on the current
    device, and what is left of their scales; returns (the memory that holds them, the addresses
    of the K pages, of the V pages and of the factors in it, the identity page table's memory and
    its columns, pages).  The memory belongs to the call: what another thread enqueues between the
    two launches, on this stream too, has its own.  torch's allocator hands it out again in stream
    order only."""
    nb, nkv, bs, hd = k_cache.shape
    width = page_table.shape[1]
    capturing = torch.cuda.is_current_stream_capturing()
    if max_context_len < 0:
        raise ValueError("max_context_len must not be negative")
    if capturing:
        max_context_len = 0
    if max_context_len > 0:
        width = min(width, (max_context_len + bs - 1) // bs)
    pages = max(num_seqs * width, 1)
    dev = k_cache.device
    stream = _raw_stream(dev.index)
    half = pages * nkv * bs * hd * 2
    pool = k_cache.new_empty(2 * half + pages * nkv * 8)         # elements of one byte
    k_pool = pool.data_ptr()
    v_pool, factors = k_pool + half, k_pool + 2 * half
    _lib.check(
        "b200attn_dequant_pages_scaled_ex",
        _lib.lib().b200attn_dequant_pages_scaled_ex(
            k_pool, v_pool, factors, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), _cache_dtype(k_cache), page_table.data_ptr(), page_table.stride(0),
            width, cu_q.data_ptr(), q_start.data_ptr() if q_start is not None else 0,
            max_context_len, num_seqs, nkv, hd, bs, nb, stream))
    return pool, k_pool, v_pool, factors, _identity_table(dev, stream, pages, capturing), width, pages


def read_error_word(device: Optional[torch.device] = None) -> int:
    """Returns and clears the device diagnostics word (0 = clean, 1 = a bounded wait ran out,
    2 = a page id or slot pointed outside the cache)."""
    word = ctypes.c_int32(0)
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    with torch.cuda.device(dev):
        _lib.check(
            "b200attn_read_error_word",
            _lib.lib().b200attn_read_error_word(
                ctypes.byref(word), torch.cuda.current_stream(dev).cuda_stream
            ),
        )
    if word.value:
        # an aborted launch may have left arrival counters behind: start the scratch afresh
        for ws in list(_workspaces.values()) + _retired_workspaces:
            if ws.device == dev:
                ws[:TICKET_BYTES].zero_()
    return int(word.value)


class ErrorWordWatch:
    """Once-per-step watch on the device diagnostics word for a serving loop.  `poll()` raises if
    an EARLIER poll's asynchronous copy found the word set, then queues the next copy on the
    current stream; it never synchronises.  A kernel that gave up on a bounded wait (word 1) or
    met a page id outside the cache (word 2) is therefore reported a step or two later instead
    of passing silently."""

    MESSAGES = {
        1: "a bounded wait inside a b200attn kernel ran out (diagnostics word 1): outputs of the "
           "launches around it are invalid; a row-parallel communicator involved must be rebuilt",
        2: "a page id or slot outside the KV cache reached a b200attn kernel (diagnostics word 2): "
           "the access was skipped; the step's metadata is inconsistent with the cache",
    }

    # called with the word's value before poll() raises (e.g. to switch a fused path off)
    on_error: list = []

    def __init__(self, device: Optional[torch.device] = None):
        self.device = device if device is not None else torch.device(
            "cuda", torch.cuda.current_device())
        self._host = torch.zeros(1, dtype=torch.int32)
        if torch.cuda.is_available():
            self._host = self._host.pin_memory()

    def value(self) -> int:
        return int(self._host[0])

    def poll(self) -> None:
        word = self.value()
        if word:
            self._host.zero_()
            for react in list(self.on_error):
                react(word)
            if self.device.type == "cuda" and torch.cuda.is_available():
                read_error_word(self.device)      # clear on the device too
            raise RuntimeError(self.MESSAGES.get(word, f"device diagnostics word {word}"))
        _lib.check(
            "b200attn_peek_error_word_async",
            _lib.lib().b200attn_peek_error_word_async(
                self._host.data_ptr(), torch.cuda.current_stream(self.device).cuda_stream),
        )
