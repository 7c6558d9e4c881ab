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
_DTYPE_CODES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_FP16}


# A small step's launches take a few microseconds each, so the checks below ask
# each tensor little and look closer only to name what is wrong.


def _misplaced(tensor: torch.Tensor, name: str, like: torch.Tensor) -> ValueError:
    dev.require_hip(like, "the step's tensors")
    dev.require_hip(tensor, name)
    return ValueError(f"{name} is on {tensor.device}, the step's other tensors are on {like.device}")


def _call(device: torch.device, name: str, *args: object) -> None:
    """Launch on the device's current stream, with the device current."""
    if device.index is None or device.index == torch.cuda.current_device():
        _native.call(name, dev.stream_handle(device), *args)
    else:
        with torch.cuda.device(device):
            _native.call(name, dev.stream_handle(device), *args)


def _vector(tensor: torch.Tensor, name: str, dtype: torch.dtype, like: torch.Tensor, where: int, length: int | None = None) -> int:
    """A contiguous vector on ``like``'s device, whose number is ``where``; returns its address."""
    if (
        tensor.dtype is dtype
        and tensor.get_device() == where
        and tensor.dim() == 1
        and tensor.is_contiguous()
        and (length is None or tensor.numel() == length)
    ):
        return tensor.data_ptr()
    if tensor.get_device() != like.get_device():
        raise _misplaced(tensor, name, like)
    dev.require_dtype(tensor, name, dtype)
    if tensor.dim() != 1 or not tensor.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector")
    raise ValueError(f"{name} must have {length} entries, got {tensor.numel()}")


def _block_table(table: torch.Tensor, n: int, like: torch.Tensor) -> tuple[int, int]:
    """(row stride, blocks a row) of an int32 table with a row for each of n requests."""
    if table.get_device() != like.get_device():
        raise _misplaced(table, "block_table", like)
    if table.dtype is not torch.int32:
        dev.require_dtype(table, "block_table", torch.int32)
    if table.dim() != 2:
        raise ValueError("block_table must be [requests, max_blocks] with contiguous rows")
    (rows, blocks), (stride, inner) = table.shape, table.stride()
    if rows < n or (blocks > 1 and inner != 1):
        raise ValueError("block_table must be [requests, max_blocks] with contiguous rows and a row for every request")
    return (stride if rows > 1 else blocks), blocks


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
    No written tensor may overlap another of the call's.
    ``max_query_len`` (the longest request's new tokens, if the host knows it)
    only sizes the launch."""
    dev.require_hip(computed_tokens, "computed_tokens")
    like, where, n = computed_tokens, computed_tokens.get_device(), computed_tokens.numel()
    computed = _vector(computed_tokens, "computed_tokens", torch.int32, like, where)
    new = _vector(new_tokens, "new_tokens", torch.int32, like, where, n)
    offsets = None if request_offsets is None else _vector(request_offsets, "request_offsets", torch.int64, like, where, n)
    ids = _vector(block_ids, "block_ids", torch.int64, like, where)
    id_offsets = _vector(block_offsets, "block_offsets", torch.int64, like, where, n + 1)
    start = _vector(query_start_loc, "query_start_loc", torch.int32, like, where, n + 1)
    lens = _vector(seq_lens, "seq_lens", torch.int32, like, where)
    if seq_lens.numel() < n:
        raise ValueError("seq_lens must have an entry for every request")
    tokens = positions.numel()
    places = _vector(positions, "positions", torch.int64, like, where)
    slots = _vector(slot_mapping, "slot_mapping", torch.int64, like, where, tokens)
    stride, blocks = _block_table(block_table, n, like)
    longest = tokens if max_query_len is None else int(max_query_len)
    if longest < 0:
        raise ValueError("max_query_len must be non-negative")
    _call(
        like.device, "kvc_step_tables", n, computed, new, offsets, ids, id_offsets, int(page_tokens), longest, tokens, blocks, stride, start,
        lens, places, slots, block_table.data_ptr(),
    )


# ------------------------------------------------------------------ rotary --


def _heads(tensor: torch.Tensor, name: str, tokens: int, like: torch.Tensor) -> tuple[int, int, int, int]:
    """[tokens, heads, D] of the cache ``like`` with unit inner stride: (address,
    token stride, head stride, heads); a dimension of one entry has no stride."""
    if tensor.get_device() != like.get_device():
        raise _misplaced(tensor, name, like)
    shape, dim = tensor.shape, like.shape[3]
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim:
        raise ValueError(f"{name} must have shape [{tokens}, heads, {dim}], got {tuple(shape)}")
    if tensor.dtype is not like.dtype:
        raise ValueError(f"{name} must have the cache's dtype {like.dtype}, got {tensor.dtype}")
    token, head, inner = tensor.stride()
    if inner != 1:
        raise ValueError(f"{name} must have contiguous heads")
    return tensor.data_ptr(), (token if tokens > 1 else 0), (head if shape[1] > 1 else 0), shape[1]


def _cache_pair(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(dtype code, pages, page stride, KV heads, head dim) of the two caches."""
    dev.require_hip(k_cache, "k_cache")
    code, shape, step = _DTYPE_CODES.get(k_cache.dtype), k_cache.shape, k_cache.stride()
    if code is None or len(shape) != 4:
        dev.validate_cache(k_cache, "k_cache")
    pages, block, heads, dim = shape
    row = heads * dim
    if block != dev.BLOCK_SIZE or step[1:] != (row, dim, 1) or step[0] < block * row:
        dev.validate_cache(k_cache, "k_cache")
    if v_cache.get_device() != k_cache.get_device():
        raise _misplaced(v_cache, "v_cache", k_cache)
    if v_cache.dtype is not k_cache.dtype or v_cache.shape != shape or v_cache.stride() != step:
        raise ValueError("K and V caches must share shape, strides and dtype")
    return code, pages, step[0], heads, dim


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
    store nothing.  Returns the rotated queries: ``q_out`` or a new tensor;
    ``q_out`` may be ``q``, but overlap no other of the step's tensors."""
    code, pages, page_stride, kv_heads, dim = _cache_pair(k_cache, v_cache)
    tokens = slot_mapping.numel()
    where = k_cache.get_device()
    slots = _vector(slot_mapping, "slot_mapping", torch.int64, k_cache, where)
    *q_place, heads = _heads(q, "q", tokens, k_cache)
    *k_place, k_heads = _heads(k, "k", tokens, k_cache)
    *v_place, v_heads = _heads(v, "v", tokens, k_cache)
    if k_heads != kv_heads or v_heads != kv_heads:
        raise ValueError(f"{'v' if k_heads == kv_heads else 'k'} must have the cache's {kv_heads} heads")
    if q_out is None:
        q_out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    *out_place, out_heads = _heads(q_out, "q_out", tokens, k_cache)
    if out_heads != heads:
        raise ValueError("q_out must have q's heads")
    if heads and out_place[0] == q_place[0] and out_place != q_place:
        raise ValueError("q_out may be q itself, but not another view of it")
    freq = omega.numel()
    turns = _vector(omega, "omega", torch.float32, k_cache, where)
    if not 0 < 2 * freq <= dim:
        raise ValueError(f"omega must hold one to head_dim/2 = {dim // 2} frequencies, got {freq}")
    if positions.get_device() != k_cache.get_device():
        raise _misplaced(positions, "positions", k_cache)
    if positions.dtype is not torch.int64:
        dev.require_dtype(positions, "positions", torch.int64)
    shape, step = positions.shape, positions.stride()
    if not 1 <= len(shape) <= 2 or shape[-1] != tokens or (tokens > 1 and step[-1] != 1):
        raise ValueError("positions must be [tokens] or [axes, tokens] with contiguous rows")
    axes, axis_step = (1, 0) if len(shape) == 1 else (shape[0], step[0])
    share = (freq,) if sections is None else tuple(int(x) for x in sections)
    if not 1 <= axes <= 4 or len(share) != axes:
        raise ValueError(f"sections must name the frequencies of each of the {axes} axes (one to four)")
    if min(share) < 0 or sum(share) != freq:
        raise ValueError(f"sections {share} must be non-negative and add up to {freq} frequencies")
    if axis_order not in AXIS_ORDERS:
        raise ValueError(f"axis_order must be one of {', '.join(AXIS_ORDERS)}, got {axis_order!r}")
    _call(
        k_cache.device, "kvc_rotate_and_store", code, dev.rope_style_code(rope_style), tokens, heads, kv_heads,
        dim, 2 * freq, *q_place, *k_place, *v_place, positions.data_ptr(), axis_step, axes, (ctypes.c_int * axes)(*share),
        int(axis_order == "cycled"), turns, slots, *out_place, k_cache.data_ptr(), v_cache.data_ptr(), pages, page_stride,
    )
    return q_out


# --------------------------------------------------------------- attention --


def attend_workspace_bytes(
    heads: int, kv_heads: int, head_dim: int, n_seq: int, num_tokens: int, max_query_len: int, max_seq_len: int
) -> int:
    """Bytes of :func:`attend_paged`'s workspace for a step of these sizes, and for
    any with none of the last four larger."""
    if kv_heads <= 0 or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the KV heads")
    size = _native.load().kvc_attend_workspace_bytes(kv_heads, heads // kv_heads, head_dim, n_seq, num_tokens, max_query_len, max_seq_len)
    if size == 0:
        raise ValueError(
            f"unsupported attention shape (head_dim {head_dim} must be a multiple of 8 up to 256, tokens {num_tokens} below 2^24, "
            f"tokens x query heads of a KV head below 2^31 - 256)"
        )
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
    may not overlap q or hold a row twice; rows outside every request are not
    written.
    ``workspace``: uint8, at least :func:`attend_workspace_bytes`, for callers
    that keep one per stream; calls that overlap in time need one each."""
    code, pages, page_stride, kv_heads, dim = _cache_pair(k_cache, v_cache)
    tokens = q.shape[0]
    *q_place, heads = _heads(q, "q", tokens, k_cache)
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a positive multiple of the cache's KV heads ({kv_heads})")
    n = query_start_loc.numel() - 1
    where = k_cache.get_device()
    start = _vector(query_start_loc, "query_start_loc", torch.int32, k_cache, where)
    if n < 0:
        raise ValueError("query_start_loc must have one entry more than there are requests")
    lens = _vector(seq_lens, "seq_lens", torch.int32, k_cache, where)
    if seq_lens.numel() < n:
        raise ValueError("seq_lens must have a row for every request")
    stride, blocks = _block_table(block_table, n, k_cache)
    longest = tokens if max_query_len is None else min(int(max_query_len), tokens)
    reach = blocks * dev.BLOCK_SIZE if max_seq_len is None else min(int(max_seq_len), blocks * dev.BLOCK_SIZE)
    if longest < 0 or reach < 0:
        raise ValueError("max_query_len and max_seq_len must be non-negative")
    factor = dim**-0.5 if scale is None else float(scale)
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError("scale must be positive and finite")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must be non-negative")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    *out_place, out_heads = _heads(out, "out", tokens, k_cache)
    if out_heads != heads:
        raise ValueError("out must have q's shape")
    size = attend_workspace_bytes(heads, kv_heads, dim, n, tokens, longest, reach)
    if workspace is None:
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != k_cache.get_device():
        raise _misplaced(workspace, "workspace", k_cache)
    elif not workspace.is_contiguous() or workspace.nbytes < size:
        raise ValueError(f"workspace must be contiguous and hold at least {size} bytes")
    most = (1 << 31) - 1
    _call(
        k_cache.device, "kvc_attend_paged", code, *q_place, k_cache.data_ptr(), v_cache.data_ptr(), pages,
        page_stride, kv_heads, heads // kv_heads, dim, n, tokens, start, lens, block_table.data_ptr(), stride, blocks, longest, reach,
        factor, min(int(window), most), min(int(sinks), most), *out_place, workspace.data_ptr(), workspace.nbytes,
    )
    return out
