"""Paged K/V cache: block tables, appends and attention for ragged batches.

The segmented cache (segmented_cache.py) holds one lockstep batch in packed
slabs.  For requests of different lengths that come and go, and for batches
that share a prompt, K/V rows live in blocks ``[num_blocks, kv_heads,
block_size, D]`` and each request has a table of its blocks.  One step of a
batch is

* :func:`build_paged_tables`, once: blocks taken from and given back to a ring
  of free ones, block tables, slot map and query starts, all on the GPU;
* per layer :func:`append_paged_kv` (the step's K/V rows to their slots) and
  :func:`paged_window_attention` or :func:`paged_shared_prefix_attention`.

No step reads anything back to the host, so a step can be captured in a HIP
graph and replayed.  Inference only, as the rest of the package: nothing here
has a gradient, and inputs that require one are refused while grad mode is on.
The reference has no counterpart: its cache is one lockstep batch
(enable_real_pruning_fast.py:1951-2254).
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_REQUESTS = 4096
HEAD_DIMS = (64, 128)
MAX_BLOCK_SIZE = 1 << 20


class PagedStep(NamedTuple):
    """What :func:`build_paged_tables` gives for one step."""

    slot_map: torch.Tensor
    query_starts: torch.Tensor
    lengths: torch.Tensor
    free_range: torch.Tensor
    status: torch.Tensor


def _check_block_size(block_size: int) -> int:
    block_size = int(block_size)
    if block_size <= 0 or block_size & (block_size - 1) or block_size > MAX_BLOCK_SIZE:
        raise ValueError(f"block_size must be a power of two up to 2^20 (got {block_size})")
    return block_size


def _check_window(window: int, sinks: int):
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0 or window >= 2**31 or sinks >= 2**31:
        raise ValueError(f"window and sinks must lie in [0, 2^31) (got {window}, {sinks})")
    return window, sinks


def _check_ints(what: str, t: torch.Tensor, shape, device) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be an int32 tensor {list(shape)} (got {t.dtype} {list(t.shape)})")
    if t.device != device:
        raise ValueError(f"{what} must be on {device} (got {t.device})")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _check_table(block_tables: torch.Tensor) -> None:
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2:
        raise ValueError("block_tables must be an int32 tensor [R, M]")
    if block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables must have contiguous rows")
    if block_tables.shape[0] > 1 and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError("block_tables must not have rows that overlap")
    if block_tables.shape[0] > MAX_REQUESTS:
        raise RuntimeError(f"the paged cache takes at most {MAX_REQUESTS} requests (got {block_tables.shape[0]})")


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or detach its inputs")


def _check_caches(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor):
    """Shape ``(num_blocks, kv_heads, block_size, D)`` of the two caches."""
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must be [num_blocks, kv_heads, block_size, D] tensors of one shape")
    if v_cache.dtype != k_cache.dtype or v_cache.device != k_cache.device:
        raise ValueError("k_cache and v_cache must share dtype and device")
    if k_cache.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"{what} takes float16 or bfloat16 caches (got {k_cache.dtype})")
    n, heads, block, dim = (int(x) for x in k_cache.shape)
    if dim not in HEAD_DIMS:
        raise RuntimeError(f"{what} takes head_dim 64 or 128 (got {dim})")
    if heads == 0:
        raise ValueError("the caches must have at least one K/V head")
    if n >= 2**31:
        raise RuntimeError(f"{what} takes fewer than 2^31 blocks (got {n})")
    _check_block_size(block)
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the rows of k_cache and v_cache must be contiguous")
    return n, heads, block, dim


def _call(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` on ``device``'s current stream, ``device`` made current for the launch."""
    if device.index is not None and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def build_paged_tables(
    *,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    new_counts: torch.Tensor,
    free_blocks: torch.Tensor,
    free_range: torch.Tensor,
    num_tokens: int,
    block_size: int,
    window: int = 0,
    sinks: int = 0,
    in_place: bool = False,
) -> PagedStep:
    """One step's bookkeeping of a paged cache, on the GPU.

    * ``block_tables`` int32 ``[R, M]`` (written in place): block ids of each
      request in order; ``lengths`` int32 ``[R]``: rows each holds;
    * ``new_counts`` int32 ``[R]``: tokens each brings (0: none; negative: the
      request has ended and gives its blocks back);
    * ``free_blocks`` int32 ``[N]`` (written in place), ``free_range`` int32
      ``[2]``: a ring of free block ids and its (first, count).  N is at least
      the number of blocks that can be free at once;
    * ``num_tokens``: the step's tokens, or more (a padded batch);
    * ``window``, ``sinks``: as the attention's (0: no window).  Blocks that
      have left the window, behind the first ``sinks`` rows' blocks, are given
      back too; their table entries keep their values and are not read again.
      Every step of a cache passes the same two values.

    Blocks are taken from the ring's head in request order; blocks given back
    follow its tail in request and table order and are taken by later steps
    only, so this step's attention may still read them.

    Returns ``slot_map`` int64 ``[num_tokens]`` (block * block_size + row of
    each token, requests back to back, -1 behind the last), ``query_starts``
    int32 ``[R + 1]``, the new ``lengths`` and ``free_range`` (new tensors, or
    with ``in_place`` the given ones, updated) and ``status`` int32 ``[1]``: 0,
    or a sum of 1 (too few free blocks), 2 (a request does not fit its table
    row) and 4 (more tokens than ``num_tokens``), or 8 (more blocks given back
    than the ring has room for).  A step with a nonzero status changes nothing:
    every slot is -1, every query start 0, and the state is as before.
    Calling it again with the same inputs gives the same results
    (unless ``in_place``).
    """
    native = _lib.op_call
    if native is not None:
        got = native.paged_tables(block_tables, lengths, new_counts, free_blocks, free_range, num_tokens, block_size,
                                  window, sinks, in_place)
        if got is not None:
            return PagedStep._make(got)
    _check_table(block_tables)
    R, M = (int(x) for x in block_tables.shape)
    device = block_tables.device
    _check_ints("lengths", lengths, (R,), device)
    _check_ints("new_counts", new_counts, (R,), device)
    _check_ints("free_range", free_range, (2,), device)
    if free_blocks.ndim != 1:
        raise ValueError("free_blocks must be an int32 tensor [N]")
    _check_ints("free_blocks", free_blocks, (int(free_blocks.shape[0]),), device)
    num_tokens = int(num_tokens)
    if num_tokens < 0 or num_tokens >= 2**31:
        raise ValueError(f"num_tokens must lie in [0, 2^31) (got {num_tokens})")
    block_size = _check_block_size(block_size)
    window, sinks = _check_window(window, sinks)
    if device.type != "cuda":
        raise RuntimeError("build_paged_tables requires CUDA tensors")
    _lib.require_device(device)
    slot_map = torch.empty((num_tokens,), dtype=torch.int64, device=device)
    query_starts = torch.empty((R + 1,), dtype=torch.int32, device=device)
    status = torch.empty((3,), dtype=torch.int32, device=device)
    lengths_out = lengths if in_place else torch.empty_like(lengths)
    range_out = free_range if in_place else torch.empty_like(free_range)
    _call(device, _lib.load().hkv_paged_tables, block_tables.data_ptr(), int(block_tables.stride(0)),
          lengths.data_ptr(), new_counts.data_ptr(), free_blocks.data_ptr(), free_range.data_ptr(), R, M,
          int(free_blocks.shape[0]), num_tokens, block_size, window, sinks, slot_map.data_ptr(),
          query_starts.data_ptr(), lengths_out.data_ptr(), range_out.data_ptr(), status.data_ptr())
    return PagedStep(slot_map, query_starts, lengths_out, range_out, status[:1])


def append_paged_kv(
    *,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_map: torch.Tensor,
):
    """Writes K/V rows ``[T, kv_heads, D]`` to their slots of the paged cache
    in place; returns ``(k_cache, v_cache)``.

    ``slot_map`` int64 ``[T]`` (:func:`build_paged_tables`): block * block_size
    + row, distinct; tokens whose slot lies outside the cache (-1) are skipped.
    k and v may have any token and head strides (rows contiguous), the caches
    any block, head and row strides: ``[N, block, kv_heads, D]`` storage is
    passed as ``cache.transpose(1, 2)``.
    """
    native = _lib.op_call
    if native is not None and native.paged_append(k, v, k_cache, v_cache, slot_map):
        return k_cache, v_cache
    n, heads, block, dim = _check_caches("append_paged_kv", k_cache, v_cache)
    for what, t in (("k", k), ("v", v)):
        if t.ndim != 3 or tuple(t.shape[1:]) != (heads, dim) or t.shape[0] != k.shape[0]:
            raise ValueError(f"{what} must be [T, {heads}, {dim}] (got {list(t.shape)})")
        if t.dtype != k_cache.dtype or t.device != k_cache.device:
            raise ValueError(f"{what} must share the caches' dtype and device")
        if t.stride(2) != 1:
            raise ValueError(f"the rows of {what} must be contiguous")
    T = int(k.shape[0])
    if slot_map.dtype != torch.int64 or tuple(slot_map.shape) != (T,) or slot_map.device != k_cache.device:
        raise ValueError(f"slot_map must be an int64 tensor [{T}] on the caches' device")
    if not slot_map.is_contiguous():
        raise ValueError("slot_map must be contiguous")
    if k_cache.device.type != "cuda":
        raise RuntimeError("append_paged_kv requires CUDA tensors")
    if T >= 2**31:
        raise RuntimeError(f"append_paged_kv takes fewer than 2^31 tokens (got {T})")
    _no_grad("append_paged_kv", k, v, k_cache, v_cache)
    _lib.require_device(k_cache.device)
    _call(k_cache.device, _lib.load().hkv_paged_append, k.data_ptr(), v.data_ptr(), int(k.stride(0)),
          int(k.stride(1)), int(v.stride(0)), int(v.stride(1)), k_cache.data_ptr(), v_cache.data_ptr(),
          *(int(x) for x in k_cache.stride()[:3]), *(int(x) for x in v_cache.stride()[:3]), slot_map.data_ptr(),
          n, T, heads, dim, block)
    return k_cache, v_cache


def _attention(name, q, k_cache, v_cache, prefix_blocks, prefix_length, block_tables, lengths, query_starts,
               softmax_scale, window, sinks, causal, out, return_lse):
    native = _lib.op_call
    if native is not None:
        got = native.paged_attention(q, k_cache, v_cache, prefix_blocks, prefix_length, block_tables, lengths,
                                     query_starts, softmax_scale, window, sinks, causal, out, return_lse)
        if got is not None:
            return got
    n, kv_heads, block, dim = _check_caches(name, k_cache, v_cache)
    device = k_cache.device
    if q.ndim != 3 or int(q.shape[2]) != dim:
        raise ValueError(f"q must be [T, H, {dim}] (got {list(q.shape)})")
    if q.dtype != k_cache.dtype or q.device != device:
        raise ValueError("q must share the caches' dtype and device")
    T, heads = int(q.shape[0]), int(q.shape[1])
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"q's heads must be a multiple of the {kv_heads} K/V heads (got {heads})")
    if heads > 1024:
        raise RuntimeError(f"{name} takes at most 1024 heads (got {heads})")
    _check_table(block_tables)
    R, M = (int(x) for x in block_tables.shape)
    if block_tables.device != device:
        raise ValueError(f"block_tables must be on {device} (got {block_tables.device})")
    _check_ints("lengths", lengths, (R,), device)
    _check_ints("query_starts", query_starts, (R + 1,), device)
    window, sinks = _check_window(window, sinks)
    softmax_scale = float(softmax_scale)
    if not math.isfinite(softmax_scale):
        raise ValueError(f"softmax_scale must be finite (got {softmax_scale})")
    prefix_length = int(prefix_length)
    if prefix_length < 0 or prefix_length >= 2**31:
        raise ValueError(f"prefix_length must lie in [0, 2^31) (got {prefix_length})")
    if prefix_blocks is not None:
        if prefix_blocks.ndim != 1:
            raise ValueError("prefix_blocks must be an int32 tensor [P]")
        _check_ints("prefix_blocks", prefix_blocks, (int(prefix_blocks.shape[0]),), device)
        if prefix_length > int(prefix_blocks.shape[0]) * block:
            raise ValueError(f"prefix_blocks hold {int(prefix_blocks.shape[0]) * block} rows, "
                             f"prefix_length is {prefix_length}")
    if n == 0 and (M > 0 or prefix_length > 0):
        raise ValueError("the cache has no blocks")
    if out is not None:
        if tuple(out.shape) != (T, heads * dim) or out.dtype != q.dtype or out.device != device:
            raise ValueError(f"out must be [{T}, {heads * dim}] of q's dtype and device")
        if not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous and start on a 16-byte boundary")
    if device.type != "cuda":
        raise RuntimeError(f"{name} requires CUDA tensors")
    for what, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]):
            raise ValueError(f"{what} must start, and its rows lie, on 16-byte boundaries")
    _no_grad(name, q, k_cache, v_cache)
    _lib.require_device(device)
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    fill = out is None
    if fill:
        out = torch.empty((T, heads * dim), dtype=q.dtype, device=device)
    lse = torch.empty((heads, T), dtype=torch.float32, device=device) if return_lse else None
    lib = _lib.load()
    need = int(lib.hkv_paged_attention_workspace_bytes(T, R, heads, kv_heads, dim, M, block, prefix_length,
                                                       window, sinks, 1 if causal else 0))
    _lib.check(min(need, 0))
    ws = torch.empty((need,), dtype=torch.uint8, device=device) if need > 0 else None
    _call(device, lib.hkv_paged_attention, q.data_ptr(), int(q.stride(0)), int(q.stride(1)), k_cache.data_ptr(),
          v_cache.data_ptr(), *(int(x) for x in k_cache.stride()[:3]), *(int(x) for x in v_cache.stride()[:3]),
          block_tables.data_ptr(), int(block_tables.stride(0)), lengths.data_ptr(), query_starts.data_ptr(),
          prefix_blocks.data_ptr() if prefix_length > 0 else None, prefix_length, out.data_ptr(),
          lse.data_ptr() if lse is not None else None, T, R, M, n, heads, kv_heads, dim, block, window, sinks,
          1 if causal else 0, _lib.dtype_code(q.dtype), softmax_scale, 1 if fill else 0,
          ws.data_ptr() if ws is not None else None, need,
          _lib.paged_counters(device).data_ptr() if need > 0 else None)
    return (out, lse) if return_lse else out


def paged_window_attention(
    *,
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    query_starts: torch.Tensor,
    softmax_scale: float,
    window: int = 0,
    sinks: int = 0,
    causal: bool = True,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """Attention of each request's new tokens over its rows of the paged cache.

    * ``q`` ``[T, H, D]`` (bf16 or fp16, D 64 or 128; any token and head
      strides): the requests' queries back to back, request r's at
      ``query_starts[r] .. query_starts[r + 1]`` (int32 ``[R + 1]``);
    * ``k_cache``, ``v_cache`` ``[N, kv_heads, block_size, D]`` of q's dtype,
      any block, head and row strides that keep rows on 16-byte boundaries; H
      is a multiple of kv_heads and query head h reads K/V head
      ``h // (H // kv_heads)``;
    * ``block_tables`` int32 ``[R, M]``, ``lengths`` int32 ``[R]``: each
      request's blocks and its rows, this step's included.

    The n queries of a request are its last n rows: query i stands at row
    ``p = length - n + i``.  It sees row j if ``j <= p`` (``causal``; without it
    every row of the request, as the tokens of one scale see each other) and,
    with ``window`` > 0, ``j > p - window`` or ``j < sinks``: the last
    ``window`` rows up to its own and the first ``sinks`` ones.  Rows that no
    query of the request sees are not read, nor their table entries.  Values
    that a query does not see (infinities and NaN included) have no effect on
    it.  A query that stands before row 0 sees nothing; such queries get zeros
    (lse -inf).  Lengths beyond the table's rows count as those, and table
    entries that name no block of the cache stand for block 0.

    Returns ``[T, H * D]`` in q's dtype and, with ``return_lse``, the fp32
    log-sum-exp ``[H, T]``.  Tokens outside the requests' (before
    ``query_starts[0]``, behind ``query_starts[R]``) get zeros (lse -inf); with
    ``out`` (``[T, H * D]``, contiguous) they keep what it held.

    Weights are rounded to q's 16-bit type for their product with V, as the
    segmented attention's are; scores, maxima, sums and accumulators are fp32.
    """
    return _attention("paged_window_attention", q, k_cache, v_cache, None, 0, block_tables, lengths, query_starts,
                      softmax_scale, window, sinks, causal, out, return_lse)


def paged_shared_prefix_attention(
    *,
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    prefix_blocks: torch.Tensor,
    prefix_length: int,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    query_starts: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """:func:`paged_window_attention` for requests that share a prefix.

    Every query sees the first ``prefix_length`` rows of ``prefix_blocks``
    (int32 ``[P]``, blocks of the same cache) and, as there, its request's own
    rows, which follow them: ``block_tables`` and ``lengths`` count a request's
    own rows only.  The prefix is read once for the queries of all requests
    together (a system prompt, or the early scales of images that continue
    differently), not once per request.
    """
    if prefix_blocks is None:
        raise ValueError("prefix_blocks must be an int32 tensor [P]")
    return _attention("paged_shared_prefix_attention", q, k_cache, v_cache, prefix_blocks, prefix_length,
                      block_tables, lengths, query_starts, softmax_scale, 0, 0, causal, out, return_lse)
