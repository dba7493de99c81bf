"""Block tables and slot maps built on the GPU from request lengths: the step
between a scheduler and append_kv() / decode(), without a trip to the host.

A pool of pages is a stack: `free_pages` int32 [capacity] holds the free page
ids in its first `free_count` (int32 [1], on the device) entries.
plan_append() takes pages from its top, release_pages() pushes them back.
Both enqueue one kernel on the current stream.  No counterpart in the
reference (its adapters build block tables on the host,
decodebench/flashinfer_kernel.py:65-92).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .api import B2DError, DecodeWorkspace, _ptr
from .ragged import _ints, _on, _one_device, _stream, _table, _workspace


class AppendPlan(NamedTuple):
    slot_mapping: torch.Tensor    # int64 [max_tokens], for append_kv()
    query_starts: torch.Tensor    # int32 [B + 1], first new token of each request
    cache_seqlens: torch.Tensor   # int32 [B], lengths after the step
    free_count: torch.Tensor      # int32 [1]


def _pool(where: str, cache_seqlens, block_table, free_pages, free_count, page_size) -> int:
    if not cache_seqlens.is_cuda:
        raise RuntimeError(f"b200decode.{where} needs CUDA tensors (there is no CPU path)")
    bsz = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else -1
    _ints(where, "cache_seqlens", cache_seqlens, bsz)
    _ints(where, "free_count", free_count, 1)
    _table(where, "block_table", block_table, bsz)
    if bsz > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError(f"{where}: block_table rows overlap")
    if free_pages.dim() != 1:
        raise ValueError(f"{where}: free_pages must be contiguous int32 [capacity]")
    _ints(where, "free_pages", free_pages, free_pages.shape[0])
    if page_size <= 0:
        raise ValueError(f"{where}: page_size must be positive")
    return bsz


def _check_out(where: str, name: str, t: torch.Tensor, n: int, dtype: torch.dtype) -> None:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{where}: {name} must be contiguous {dtype} [{n}]")


_HEADER = _lib.B2D_WORKSPACE_HEADER_BYTES


def plan_append(cache_seqlens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                free_count: torch.Tensor, page_size: int, *, new_tokens: Optional[torch.Tensor] = None,
                max_tokens: Optional[int] = None, slot_mapping: Optional[torch.Tensor] = None,
                query_starts: Optional[torch.Tensor] = None, seqlens_out: Optional[torch.Tensor] = None,
                free_count_out: Optional[torch.Tensor] = None,
                workspace: Optional[DecodeWorkspace] = None) -> AppendPlan:
    """Room for the next tokens of every request: takes the pages they need
    from the pool, writes them into block_table (in place) and gives the slot
    of each new token for append_kv().

    cache_seqlens int32 [B]: tokens that each request holds, in the first
    ceil(len / page_size) pages of its row of block_table int32 [B,
    max_pages].  new_tokens int32 [B] (None: one each).  max_tokens: length of
    slot_mapping (default: B without new_tokens; needed with them, unless
    slot_mapping is given); entries behind the last new token are -1, which
    append_kv() skips.  The k-th new page of the step, in request then page
    order, is free_pages[free_count - 1 - k].

    seqlens_out and free_count_out may be cache_seqlens and free_count
    themselves, so that a captured step continues the last one.  A step that
    does not fit (free pages, table columns or max_tokens) changes nothing:
    slots are -1, query_starts 0, lengths and free_count as before, and
    check_device_status() raises B2D_ERR_DEVICE_CAPACITY.  A negative page taken
    from the pool gives slots of -1 and is reported (B2D_ERR_DEVICE_BOUNDS).  Up
    to 16384 requests.  In a CUDA graph, pass `workspace` to read that status.
    """
    where = "plan_append"
    bsz = _pool(where, cache_seqlens, block_table, free_pages, free_count, page_size)
    index = cache_seqlens.get_device()
    _one_device(where, index, block_table, free_pages, free_count, new_tokens, slot_mapping, query_starts,
                seqlens_out, free_count_out)
    if new_tokens is not None:
        _ints(where, "new_tokens", new_tokens, bsz)
    if max_tokens is None:
        if slot_mapping is not None:
            max_tokens = slot_mapping.shape[0]
        elif new_tokens is None:
            max_tokens = bsz
        else:
            raise ValueError(f"{where}: new_tokens needs max_tokens or slot_mapping")
    if max_tokens < 0:
        raise ValueError(f"{where}: max_tokens must not be negative")
    if slot_mapping is None:
        slot_mapping = cache_seqlens.new_empty((max_tokens,), dtype=torch.int64)
    else:
        _check_out(where, "slot_mapping", slot_mapping, max_tokens, torch.int64)
    if query_starts is None:
        query_starts = cache_seqlens.new_empty((bsz + 1,))
    else:
        _check_out(where, "query_starts", query_starts, bsz + 1, torch.int32)
    if seqlens_out is None:
        seqlens_out = torch.empty_like(cache_seqlens)
    else:
        _check_out(where, "seqlens_out", seqlens_out, bsz, torch.int32)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    else:
        _check_out(where, "free_count_out", free_count_out, 1, torch.int32)
    with _on(index):
        ws = _workspace(workspace, index, lambda: _HEADER)
        with ws.lock:
            a = _lib.PlanAppendArgs(cache_seqlens.data_ptr(), _ptr(new_tokens), block_table.data_ptr(),
                                    block_table.stride(0), free_pages.data_ptr(), free_count.data_ptr(),
                                    slot_mapping.data_ptr(), query_starts.data_ptr(), seqlens_out.data_ptr(),
                                    free_count_out.data_ptr(), bsz, block_table.shape[1], page_size, max_tokens,
                                    free_pages.shape[0], 0, ws.ptr, ws.nbytes)
            rc = _lib.load().b2d_plan_append(C.byref(a), _stream(index))
    if rc:
        raise B2DError(rc, "b2d_plan_append")
    return AppendPlan(slot_mapping, query_starts, seqlens_out, free_count_out)


def release_pages(cache_seqlens: torch.Tensor, block_table: torch.Tensor, finished: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int, *,
                  seqlens_out: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None,
                  workspace: Optional[DecodeWorkspace] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Finished requests (bool [B]) give the pages of their block_table rows
    back to the pool: pushed onto free_pages behind free_count, in request then
    page order.  Returns (cache_seqlens, free_count) after the step, the
    lengths of finished requests being 0; both may be updated in place through
    seqlens_out and free_count_out.  Keep the pages of a shared prefix out of
    the rows (as decode_shared_prefix() has them): a row's pages are given back
    once for each request that holds them.  When free_pages has no room for
    all, or a finished request is longer than its row, nothing changes and
    check_device_status() raises B2D_ERR_DEVICE_CAPACITY; when one of the pages
    is negative, B2D_ERR_DEVICE_BOUNDS (free_pages behind free_count may then
    be overwritten)."""
    where = "release_pages"
    bsz = _pool(where, cache_seqlens, block_table, free_pages, free_count, page_size)
    if finished.dtype is not torch.bool or finished.shape != (bsz,) or not finished.is_contiguous():
        raise ValueError(f"{where}: finished must be contiguous bool [{bsz}]")
    index = cache_seqlens.get_device()
    _one_device(where, index, block_table, finished, free_pages, free_count, seqlens_out, free_count_out)
    if seqlens_out is None:
        seqlens_out = torch.empty_like(cache_seqlens)
    else:
        _check_out(where, "seqlens_out", seqlens_out, bsz, torch.int32)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    else:
        _check_out(where, "free_count_out", free_count_out, 1, torch.int32)
    with _on(index):
        ws = _workspace(workspace, index, lambda: _HEADER)
        with ws.lock:
            a = _lib.ReleaseArgs(cache_seqlens.data_ptr(), finished.data_ptr(), block_table.data_ptr(),
                                 block_table.stride(0), free_pages.data_ptr(), free_count.data_ptr(),
                                 seqlens_out.data_ptr(), free_count_out.data_ptr(), bsz, block_table.shape[1],
                                 page_size, free_pages.shape[0], ws.ptr, ws.nbytes)
            rc = _lib.load().b2d_release_pages(C.byref(a), _stream(index))
    if rc:
        raise B2DError(rc, "b2d_release_pages")
    return seqlens_out, free_count_out
