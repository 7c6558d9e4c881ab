"""The model step on a paged cache that compression keeps: its tables, the
rotary positions and cache write of its tokens, and the attention that reads
the cache.

A step of a host that has no kernels of its own for these is

  build_step_tables   block table, slot mapping, positions and attention
                      lengths from the requests' lengths (the offsets of
                      compressed requests: CompressionWorker.request_offsets)
  rotate_and_store    queries and keys rotated at their semantic positions,
                      keys and values written at their physical slots
  attend_paged        the new tokens' attention over the cache

Nothing synchronises and all work is enqueued on the current stream of the
tensors' device, so a step can be captured into a graph.  Semantic positions
and physical places differ after a compaction (kernels.shift_positions):
rotations use the former, causal order, windows and sinks the latter.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch

from ... import _native
from . import _device as dev

AXIS_ORDERS = ("blocked", "cycled")


def _same_device(device: torch.device, **tensors: torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        dev.require_hip(t, name)
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the step's other tensors are on {device}")


def _call(device: torch.device, name: str, *args: object) -> None:
    """Launch on the device's current stream, with the device current."""
    if device.index is None or device.index == torch.cuda.current_device():
        _native.call(name, dev.stream_handle(device), *args)
    else:
        with torch.cuda.device(device):
            _native.call(name, dev.stream_handle(device), *args)


def _vector(tensor: torch.Tensor, name: str, dtype: torch.dtype, length: int | None = None) -> None:
    dev.require_dtype(tensor, name, dtype)
    if tensor.ndim != 1 or not tensor.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector")
    if length is not None and tensor.shape[0] != length:
        raise ValueError(f"{name} must have {length} entries, got {tensor.shape[0]}")


# ------------------------------------------------------------------ tables --


def build_step_tables(
    computed_tokens: torch.Tensor,
    new_tokens: torch.Tensor,
    request_offsets: torch.Tensor | None,
    block_ids: torch.Tensor,
    block_offsets: torch.Tensor,
    page_tokens: int,
    *,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    positions: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_table: torch.Tensor,
    max_query_len: int | None = None,
) -> None:
    """Fill a step's tables from its requests' lengths, in one launch.

    computed_tokens, new_tokens: int32 [n]; request_offsets: int64 [n] (semantic
    minus physical length, CompressionWorker.request_offsets) or None;
    block_ids/block_offsets: int64, the requests' scheduler pages of
    ``page_tokens`` tokens as one ragged table (offsets [n + 1], the form of
    pipeline.Batch).  Written: query_start_loc int32 [n + 1], seq_lens int32
    [>= n] (physical lengths after the step), positions (semantic) and
    slot_mapping int64 [tokens, padding included], block_table int32 [>= n,
    max_blocks] of 128-token pages with unit inner stride.  Entries behind a
    request's length and slots without a page are -1, padding tokens get slot
    -1 and position 0, rows of the tables behind request n stay as they were.
    ``max_query_len`` (the longest request's new tokens, if the host knows it)
    only sizes the launch."""
    device = computed_tokens.device
    _same_device(
        device, computed_tokens=computed_tokens, new_tokens=new_tokens, request_offsets=request_offsets, block_ids=block_ids,
        block_offsets=block_offsets, query_start_loc=query_start_loc, seq_lens=seq_lens, positions=positions,
        slot_mapping=slot_mapping, block_table=block_table,
    )
    _vector(computed_tokens, "computed_tokens", torch.int32)
    n = computed_tokens.shape[0]
    _vector(new_tokens, "new_tokens", torch.int32, n)
    if request_offsets is not None:
        _vector(request_offsets, "request_offsets", torch.int64, n)
    _vector(block_ids, "block_ids", torch.int64)
    _vector(block_offsets, "block_offsets", torch.int64, n + 1)
    _vector(query_start_loc, "query_start_loc", torch.int32, n + 1)
    _vector(seq_lens, "seq_lens", torch.int32)
    if seq_lens.shape[0] < n:
        raise ValueError("seq_lens must have an entry for every request")
    _vector(positions, "positions", torch.int64)
    tokens = positions.shape[0]
    _vector(slot_mapping, "slot_mapping", torch.int64, tokens)
    dev.require_dtype(block_table, "block_table", torch.int32)
    if block_table.ndim != 2 or block_table.shape[0] < n or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be [>= requests, max_blocks] with contiguous rows")
    if max_query_len is not None and max_query_len < 0:
        raise ValueError("max_query_len must be non-negative")
    _call(
        device, "kvc_step_tables", n, computed_tokens.data_ptr(), new_tokens.data_ptr(), dev.ptr(request_offsets),
        block_ids.data_ptr(), block_offsets.data_ptr(), int(page_tokens), int(tokens if max_query_len is None else max_query_len),
        tokens, block_table.shape[1], _table_stride(block_table),
        query_start_loc.data_ptr(), seq_lens.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(), block_table.data_ptr(),
    )


# ------------------------------------------------------------------ rotary --


def _heads(tensor: torch.Tensor, name: str, tokens: int, dim: int, dtype: torch.dtype) -> int:
    """[tokens, heads, dim] with unit inner stride; returns the head count."""
    if tensor.ndim != 3 or tensor.shape[0] != tokens or tensor.shape[2] != dim:
        raise ValueError(f"{name} must have shape [{tokens}, heads, {dim}], got {tuple(tensor.shape)}")
    if tensor.dtype != dtype:
        raise ValueError(f"{name} must have the cache's dtype {dtype}, got {tensor.dtype}")
    if tensor.stride(2) != 1:
        raise ValueError(f"{name} must have contiguous heads")
    return tensor.shape[1]


def _steps(tensor: torch.Tensor) -> tuple[int, int]:
    """Token and head strides; a dimension of one entry has none."""
    tokens, heads, _ = tensor.shape
    step = tensor.stride()
    return (step[0] if tokens > 1 else 0), (step[1] if heads > 1 else 0)


def _table_stride(table: torch.Tensor) -> int:
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def _cache_pair(k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    dev.validate_cache(k_cache, "k_cache")
    dev.require_hip(v_cache, "v_cache")
    if v_cache.shape != k_cache.shape or v_cache.stride() != k_cache.stride() or v_cache.dtype != k_cache.dtype:
        raise ValueError("K and V caches must share shape, strides and dtype")


def rotate_and_store(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    omega: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    sections: Sequence[int] | None = None,
    axis_order: str = "blocked",
    rope_style: str = "half",
    q_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Rotate a step's queries and keys and write keys and values to the cache.

    q [tokens, heads, D], k and v [tokens, kv_heads, D] in the cache's dtype, any
    token and head strides (parts of a fused projection are fine); omega:
    float32 [F], the angle per position of each frequency (2F rotated dims, the
    rest passes through); positions: int64 [tokens], or [axes, tokens] with
    ``sections``, the number of frequencies that each axis turns (adding up to
    F): runs of them ("blocked"), or the axes in turn while their sections
    last, what is left going with the first axis ("cycled").  ``rope_style``
    "half" pairs dims (f, F + f), "interleaved" (2f, 2f + 1).  Angles are formed
    in float64, rotations in float32, rounded once.  slot_mapping: int64
    [tokens], each slot at most once; tokens with a slot outside the cache (-1)
    store nothing.  Returns the rotated queries: ``q_out`` (may be ``q``) or a
    new tensor."""
    device = k_cache.device
    _cache_pair(k_cache, v_cache)
    _same_device(device, v_cache=v_cache, q=q, k=k, v=v, positions=positions, omega=omega, slot_mapping=slot_mapping, q_out=q_out)
    _, _, kv_heads, dim = k_cache.shape
    tokens = slot_mapping.numel()
    _vector(slot_mapping, "slot_mapping", torch.int64)
    heads = _heads(q, "q", tokens, dim, k_cache.dtype)
    for name, t in (("k", k), ("v", v)):
        if _heads(t, name, tokens, dim, k_cache.dtype) != kv_heads:
            raise ValueError(f"{name} must have the cache's {kv_heads} heads")
    if q_out is None:
        q_out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
    elif _heads(q_out, "q_out", tokens, dim, k_cache.dtype) != heads:
        raise ValueError("q_out must have q's heads")
    elif q_out.data_ptr() == q.data_ptr() and q_out.stride() != q.stride():
        raise ValueError("q_out may be q itself, but not another view of it")
    _vector(omega, "omega", torch.float32)
    freq = omega.shape[0]
    if not 0 < 2 * freq <= dim:
        raise ValueError(f"omega must hold one to head_dim/2 = {dim // 2} frequencies, got {freq}")
    dev.require_dtype(positions, "positions", torch.int64)
    if positions.ndim == 1:
        positions = positions[None]
    if positions.ndim != 2 or positions.shape[1] != tokens or (tokens > 1 and positions.stride(1) != 1):
        raise ValueError("positions must be [tokens] or [axes, tokens] with contiguous rows")
    axes = positions.shape[0]
    share = (freq,) if sections is None else tuple(int(x) for x in sections)
    if not 1 <= axes <= 4 or len(share) != axes:
        raise ValueError(f"sections must name the frequencies of each of the {axes} axes (one to four)")
    if min(share) < 0 or sum(share) != freq:
        raise ValueError(f"sections {share} must be non-negative and add up to {freq} frequencies")
    if axis_order not in AXIS_ORDERS:
        raise ValueError(f"axis_order must be one of {', '.join(AXIS_ORDERS)}, got {axis_order!r}")
    _call(
        device, "kvc_rotate_and_store", dev.cache_dtype_code(k_cache.dtype), dev.rope_style_code(rope_style), tokens, heads, kv_heads,
        dim, 2 * freq, q.data_ptr(), *_steps(q), k.data_ptr(), *_steps(k), v.data_ptr(), *_steps(v), positions.data_ptr(), positions.stride(0), axes, (ctypes.c_int * axes)(*share), int(axis_order == "cycled"),
        omega.data_ptr(), slot_mapping.data_ptr(), q_out.data_ptr(), *_steps(q_out), k_cache.data_ptr(),
        v_cache.data_ptr(), k_cache.shape[0], k_cache.stride(0),
    )
    return q_out


# --------------------------------------------------------------- attention --


def attend_workspace_bytes(
    heads: int, kv_heads: int, head_dim: int, n_seq: int, num_tokens: int, max_query_len: int, max_seq_len: int
) -> int:
    """Bytes of :func:`attend_paged`'s workspace for a step of these sizes."""
    if kv_heads <= 0 or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the KV heads")
    size = _native.load().kvc_attend_workspace_bytes(kv_heads, heads // kv_heads, head_dim, n_seq, num_tokens, max_query_len, max_seq_len)
    if size == 0:
        raise ValueError(f"unsupported attention shape (head_dim {head_dim} must be a multiple of 8 up to 256)")
    return int(size)


def attend_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    *,
    max_query_len: int | None = None,
    max_seq_len: int | None = None,
    scale: float | None = None,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a step's new tokens over the paged cache, which holds their
    own keys and values already (:func:`rotate_and_store`).

    q [tokens, heads, D] in the cache's dtype; query_start_loc int32 [n + 1],
    seq_lens int32 [>= n] (cached tokens, the new ones among them), block_table
    int32 [>= n, max_blocks] of 128-token pages: what :func:`build_step_tables`
    writes.  Token i of a request's ``new`` sits at place p = seq_len - new + i
    and sees keys j <= p; with ``window`` > 0 only those with p - j < window or
    j < ``sinks``.  Places are physical, so after a compaction a window counts
    kept tokens.  Keys in pages outside the pool are not seen, rows that see
    nothing give zeros, and a key's values never reach a row that does not see
    it.  ``max_query_len`` must bound every request's new tokens (default: all
    tokens); ``max_seq_len`` only sizes the launch (default: what the block
    table covers).  ``scale`` defaults to D ** -0.5.  ``out`` [tokens, heads, D]
    may not overlap q; rows outside every request are not written.
    ``workspace``: uint8, at least :func:`attend_workspace_bytes`, for callers
    that keep one per stream; calls that overlap in time need one each."""
    device = k_cache.device
    _cache_pair(k_cache, v_cache)
    _same_device(
        device, v_cache=v_cache, q=q, query_start_loc=query_start_loc, seq_lens=seq_lens, block_table=block_table, out=out,
        workspace=workspace,
    )
    num_pages, _, kv_heads, dim = k_cache.shape
    tokens = q.shape[0]
    heads = _heads(q, "q", tokens, dim, k_cache.dtype)
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of the cache's KV heads ({kv_heads})")
    _vector(query_start_loc, "query_start_loc", torch.int32)
    n = query_start_loc.shape[0] - 1
    if n < 0:
        raise ValueError("query_start_loc must have one entry more than there are requests")
    _vector(seq_lens, "seq_lens", torch.int32)
    dev.require_dtype(block_table, "block_table", torch.int32)
    if block_table.ndim != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be [requests, max_blocks] with contiguous rows")
    if seq_lens.shape[0] < n or block_table.shape[0] < n:
        raise ValueError("seq_lens and block_table must have a row for every request")
    max_blocks = block_table.shape[1]
    longest = tokens if max_query_len is None else int(max_query_len)
    reach = max_blocks * dev.BLOCK_SIZE if max_seq_len is None else min(int(max_seq_len), max_blocks * dev.BLOCK_SIZE)
    if longest < 0 or reach < 0:
        raise ValueError("max_query_len and max_seq_len must be non-negative")
    longest = min(longest, tokens)
    factor = dim**-0.5 if scale is None else float(scale)
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError("scale must be positive and finite")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must be non-negative")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
    elif _heads(out, "out", tokens, dim, k_cache.dtype) != heads:
        raise ValueError("out must have q's shape")
    bytes_needed = attend_workspace_bytes(heads, kv_heads, dim, n, tokens, longest, reach)
    if workspace is None:
        workspace = torch.empty(bytes_needed, dtype=torch.uint8, device=device)
    elif not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < bytes_needed:
        raise ValueError(f"workspace must be contiguous and hold at least {bytes_needed} bytes")
    most = (1 << 31) - 1
    _call(
        device, "kvc_attend_paged", dev.cache_dtype_code(k_cache.dtype), q.data_ptr(), *_steps(q), k_cache.data_ptr(),
        v_cache.data_ptr(), num_pages, k_cache.stride(0), kv_heads, heads // kv_heads, dim, n, tokens, query_start_loc.data_ptr(),
        seq_lens.data_ptr(), block_table.data_ptr(), _table_stride(block_table),
        max_blocks, longest, reach, factor, min(int(window), most), min(int(sinks), most), out.data_ptr(), *_steps(out),
        workspace.data_ptr(), workspace.numel() * workspace.element_size(),
    )
    return out
