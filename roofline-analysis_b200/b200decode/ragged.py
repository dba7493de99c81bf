"""Attention of several query tokens to one paged key sequence, and the merge
of attention states: decode over shared prefixes, cross attention to an
encoder's states, and merge_states.

Calls follow decode()'s manner (api.py): tensors on one CUDA device, work
enqueued on that device's current torch stream, no synchronisation,
ValueError for what a call cannot take and B2DError for library codes.  None
of them has a counterpart in the reference; the merge rule is
cute_attention/cluster_decode/cluster_decode_reduce.py:67-91.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Callable, Optional, Tuple

import torch

from . import _lib
from .api import _DT, B2DError, DecodeWorkspace, _check, _default_ws, _gqa_args, _ptr, _ws, decode


_stream = torch._C._cuda_getCurrentRawStream   # of a device index, without a Stream object
_here = contextlib.nullcontext()


def _on(index: int):
    """Makes device `index` the current one (nothing to do, as a rule)."""
    return _here if torch.cuda.current_device() == index else torch.cuda.device(index)


def _one_device(where: str, index: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:   # (-1: a CPU tensor)
            raise ValueError(f"{where}: all tensors must be on cuda:{index}, one is on {t.device}")


def _ints(where: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{where}: {name} must be contiguous int32 [{n}], got {t.dtype} {list(t.shape)}")


def _table(where: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] != n or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{where}: {name} must be int32 [{n}, max_pages] with contiguous rows")


def _result(where: str, name: str, t: torch.Tensor, shape, dtype: torch.dtype) -> None:
    if t.shape != shape or t.dtype is not dtype or t.stride(-1) != 1:
        raise ValueError(f"{where}: {name} must be {dtype} {list(shape)} with a contiguous last axis")


def _apart(where: str, out: torch.Tensor, q: torch.Tensor) -> None:
    # (other overlaps are the caller's to avoid; this is the likely one)
    if out.data_ptr() == q.data_ptr() and out.numel():
        raise ValueError(f"{where}: out must not be q: its rows are read until the last is written")


def _scales(where: str, hkv: int, k_scale, v_scale) -> None:
    for s in (k_scale, v_scale):
        if s is not None and (s.dtype is not torch.float32 or s.numel() != hkv or not s.is_contiguous()):
            raise ValueError(f"{where}: k_scale and v_scale must be contiguous fp32 with num_kv_heads elements")


def _workspace(workspace: Optional[DecodeWorkspace], index: int, need: Callable[[], int]) -> DecodeWorkspace:
    """The caller's workspace, or the default one of the device's current
    stream (as large as it is: the call says when that is too small).  While
    that stream is captured into a CUDA graph the default would be shared by
    every graph captured there, and could be reallocated under them: a call
    without a workspace of its own then gets one of need() bytes from the
    graph's memory pool (its header is zeroed by a node of the graph)."""
    capturing = torch.cuda.is_current_stream_capturing()
    if workspace is not None:
        if workspace.buf.get_device() != index:
            raise ValueError(f"workspace is on {workspace.buf.device}, the tensors on cuda:{index}")
        workspace.captured = workspace.captured or capturing
        return workspace.ensure(need()) if capturing else workspace.eager()
    if capturing:
        return DecodeWorkspace.in_graph(torch.device("cuda", index), need())
    return (_ws.get((index, _stream(index))) or _default_ws(torch.device("cuda", index))).eager()


def _call(fn, name: str, a, own, workspace: Optional[DecodeWorkspace], index: int, query) -> None:
    """fn(a) on the current stream, its workspace (fields of `own`) grown when
    the library finds it too small (nothing is enqueued before that check)."""
    def need() -> int:
        n = C.c_size_t(0)
        _check(query(C.byref(a), C.byref(n)), name)
        return n.value
    ws = _workspace(workspace, index, need)
    # (one call at a time: its launches hand partials to each other in the workspace)
    with ws.lock:
        buf = ws.buf
        own.workspace, own.workspace_bytes = buf.data_ptr(), buf.numel()
        rc = fn(C.byref(a), _stream(index))
        if rc == _lib.B2D_ERR_WORKSPACE:
            ws.ensure(need())
            own.workspace, own.workspace_bytes = ws.ptr, ws.nbytes
            rc = fn(C.byref(a), _stream(index))
    if rc:
        raise B2DError(rc, name)


def _caches(where: str, q: torch.Tensor, d: int, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_layout: str):
    """Checks the caches; (k strides, v strides, pages, page size, KV heads,
    layout) for the library, strides as (page, token, head)."""
    kd = k_cache.dtype
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise ValueError(f"{where}: q dtype must be bf16 or fp16, got {q.dtype}")
    if kd is not v_cache.dtype or (kd is not q.dtype and kd is not torch.float8_e4m3fn):
        raise ValueError(f"{where}: cache dtype {kd} must equal q's {q.dtype} or be float8_e4m3fn")
    shape = k_cache.shape
    if kv_layout == "vllm":
        if len(shape) != 5 or v_cache.dim() != 4 or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError(f"{where}: kv_layout='vllm' takes contiguous K [blocks, Hkv, D/x, P, x] and V "
                             "[blocks, Hkv, D, P]")
        nb, hkv, dx, page, x = shape
        if x * k_cache.element_size() != 16 or v_cache.shape != (nb, hkv, dx * x, page) or dx * x != d:
            raise ValueError(f"{where}: vLLM cache shapes do not match")
        return ((k_cache.stride(0), x, k_cache.stride(1)), (v_cache.stride(0), 1, v_cache.stride(1)),
                nb, page, hkv, _lib.B2D_KV_VLLM)
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError(f"{where}: k_cache and v_cache must be matching 4-D paged caches")
    nb, page, hkv, dc = shape
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    if dc != d:
        raise ValueError(f"{where}: head_dim mismatch between q and the caches")
    if kv_layout == "NHD":
        return ks[:3], vs[:3], nb, page, hkv, _lib.B2D_KV_STRIDED
    if kv_layout == "HND":
        return (ks[0], ks[2], ks[1]), (vs[0], vs[2], vs[1]), nb, hkv, page, _lib.B2D_KV_STRIDED
    raise ValueError(f"kv_layout must be 'NHD', 'HND' or 'vllm', got {kv_layout!r}")


def cross_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    kv_lens: torch.Tensor, block_table: torch.Tensor,
                    softmax_scale: Optional[float] = None, *,
                    query_starts: Optional[torch.Tensor] = None,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    kv_layout: str = "NHD", num_ctas: Optional[int] = None,
                    workspace: Optional[DecodeWorkspace] = None, flags: int = 0,
                    wait_limit_us: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every query token of request b attends to all kv_lens[b] states of
    request b in the paged caches (no causal mask): a decoder's cross
    attention to encoder states of another length.

    q: ragged [T, Hq, D] with query_starts int32 [B + 1] (request b owns
    tokens query_starts[b] .. query_starts[b + 1] - 1, ascending), or dense
    [B, Tq, Hq, D], or [B, Hq, D] for one token each, which is decode()'s
    kernel where that takes the sizes.  Up to 32 query heads per KV head.
    Caches, scales and layouts as in decode(); kv_lens int32 [B],
    block_table int32 [B, max_pages].  softmax_scale defaults to 1/sqrt(D).
    Returns out (shape of q) and lse (shape of q without D, fp32, natural
    log).  A request without states gives out = 0, lse = -inf; ragged tokens
    behind query_starts[B] are left as they were.  out must not overlap q.
    query_starts that descend are reported (check_device_status(),
    B2D_ERR_DEVICE_BOUNDS) and nothing is written.

    Softmax and sums are fp32; the softmax weights enter the second product
    rounded to 16 bits (the caches' type, fp16 for e4m3).  With e4m3 caches q
    enters the first product in fp16: bf16 values beyond 65504 become infinite
    (their rows NaN), those under 2^-14 lose bits.

    Captured into a CUDA graph without `workspace`, a call keeps its scratch
    in the graph's memory pool; check_device_status() reads the status only of
    a workspace that the caller passes.
    """
    where = "cross_attention"
    if not q.is_cuda:
        raise RuntimeError("b200decode.cross_attention needs CUDA tensors (there is no CPU path)")
    ragged = query_starts is not None
    dims = q.dim()
    if dims != 3 and (ragged or dims != 4):
        raise ValueError(f"{where}: q must be [T, Hq, D] with query_starts, or [B, Tq, Hq, D] or [B, Hq, D] "
                         f"without, got {tuple(q.shape)}")
    index = q.get_device()
    _one_device(where, index, k_cache, v_cache, kv_lens, block_table, query_starts, k_scale, v_scale, out, lse)
    bsz = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    _ints(where, "kv_lens", kv_lens, bsz)
    _table(where, "block_table", block_table, bsz)
    shape = q.shape
    if not ragged and shape[0] != bsz:
        raise ValueError(f"{where}: q has {shape[0]} requests, kv_lens {bsz}")
    if q.stride(-1) != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    hq, d = shape[-2:]
    ks, vs, pages, page, hkv, layout = _caches(where, q, d, k_cache, v_cache, kv_layout)
    if hq % hkv:
        raise ValueError(f"{where}: num_q_heads {hq} must be a multiple of num_kv_heads {hkv}")
    if k_scale is not None or v_scale is not None:
        _scales(where, hkv, k_scale, v_scale)
    if softmax_scale is None:
        softmax_scale = d ** -0.5
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _result(where, "out", out, shape, q.dtype)
        _apart(where, out, q)
    if lse is None:
        lse = q.new_empty(shape[:-1], dtype=torch.float32)
    else:
        _result(where, "lse", lse, shape[:-1], torch.float32)
    q3, out3, lse2, length = q, out, lse, 1
    if ragged:
        _ints(where, "query_starts", query_starts, bsz + 1)
        length = 0
    elif dims == 4:
        # [B, Tq, ...] as [B * Tq, ...]: one token stride
        length = shape[1]
        q3 = q.reshape(-1, hq, d)
        try:
            out3, lse2 = out.view(-1, hq, d), lse.view(-1, hq)
        except RuntimeError as e:
            raise ValueError(f"{where}: out and lse need one stride for all tokens") from e
    if q3.shape[0] == 0 or bsz == 0:
        return out, lse
    lib = _lib.load()
    with _on(index):
        # One token each is decode(), for the sizes that it takes (it says so before it enqueues anything).
        if length == 1 and not flags:
            try:
                ws = workspace
                if ws is not None or torch.cuda.is_current_stream_capturing():
                    g = _gqa_args(q3, k_cache, v_cache, kv_lens, block_table, softmax_scale, k_scale, v_scale, out3,
                                  lse2, kv_layout, num_ctas)
                    need = C.c_size_t(0)
                    _check(lib.b2d_gqa_workspace_bytes(C.byref(g), C.byref(need)), "b2d_gqa_workspace_bytes")
                    ws = _workspace(workspace, index, lambda: need.value)
                decode(q3, k_cache, v_cache, kv_lens, block_table, softmax_scale, k_scale=k_scale, v_scale=v_scale,
                       out=out3, lse=lse2, kv_layout=kv_layout, num_ctas=num_ctas, workspace=ws,
                       wait_limit_us=wait_limit_us)
                return out, lse
            except B2DError as e:
                if e.code != _lib.B2D_ERR_UNSUPPORTED:
                    raise
        fp8 = k_cache.dtype is torch.float8_e4m3fn
        qs, so = q3.stride(), out3.stride()
        a = _lib.CrossArgs(
            q3.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), *ks, *vs, pages,
            _ptr(query_starts), kv_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
            _ptr(k_scale) if fp8 else None, _ptr(v_scale) if fp8 else None,
            out3.data_ptr(), so[0], so[1], lse2.data_ptr(), lse2.stride(0),
            q3.shape[0], bsz, length, hq, hkv, d, page, block_table.shape[1], _DT[q.dtype], _DT[k_cache.dtype],
            softmax_scale, None, 0, num_ctas or 0, flags, layout, wait_limit_us)
        _call(lib.b2d_cross_attention, "b2d_cross_attention", a, a, workspace, index, lib.b2d_cross_workspace_bytes)
    return out, lse


def decode_shared_prefix(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         prefix_lens: torch.Tensor, prefix_block_table: torch.Tensor,
                         cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                         softmax_scale: Optional[float] = None, *,
                         group_starts: Optional[torch.Tensor] = None,
                         k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                         kv_layout: str = "NHD", num_ctas: Optional[int] = None,
                         workspace: Optional[DecodeWorkspace] = None, flags: int = 0,
                         wait_limit_us: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode() for a batch whose sequences share prefixes: sequence b attends
    to the prefix of its group and to its own tokens, and each prefix is read
    once for its whole group.

    q: [B, Hq, D] or [B, 1, Hq, D].  prefix_lens int32 [G] and
    prefix_block_table int32 [G, max_pages] describe the prefixes, cache_seqlens
    int32 [B] and block_table int32 [B, max_pages] the sequences' own tokens, all
    as pages of the same caches.  group_starts int32 [G + 1], ascending: group g
    holds sequences group_starts[g] .. group_starts[g + 1] - 1 (sequences
    outside every group have no prefix; starts that descend are reported, as in
    cross_attention()); None: one group with the whole batch.
    The rest as in decode(), whose kernels take the own tokens and whose limits
    hold here too: the query heads of a KV head split into at most 8 equal
    parts of at most 16 (8 at head_dim 192 and 256); with pages that are no
    multiples of 16, or e4m3 at head_dim 64, they are at most 8, or 16 if even;
    head_dim 192 takes 16-bit caches in pages of multiples of 16 alone.  The
    two parts, each as precise as cross_attention()'s, are joined in fp32 and
    rounded once; out must not overlap q.

    With a table whose rows begin with a common prefix of n full pages, pass
    prefix_block_table = table[:1, :n], block_table = table[:, n:] and the
    lengths minus n * P.

    Captured into a CUDA graph without `workspace`, a call keeps its scratch
    in the graph's memory pool; check_device_status() reads the status only of
    a workspace that the caller passes.
    """
    where = "decode_shared_prefix"
    if not q.is_cuda:
        raise RuntimeError("b200decode.decode_shared_prefix needs CUDA tensors (there is no CPU path)")
    index = q.get_device()
    _one_device(where, index, k_cache, v_cache, prefix_lens, prefix_block_table, cache_seqlens, block_table,
                group_starts, k_scale, v_scale, out, lse)
    groups = prefix_lens.shape[0] if prefix_lens.dim() == 1 else -1
    _ints(where, "prefix_lens", prefix_lens, groups)
    _table(where, "prefix_block_table", prefix_block_table, groups)
    if group_starts is not None:
        _ints(where, "group_starts", group_starts, groups + 1)
    elif groups > 1:
        raise ValueError(f"{where}: {groups} prefixes need group_starts")
    if q.dim() == 4 and q.shape[1] != 1:
        raise ValueError(f"{where}: one query token per sequence (q [B, 1, Hq, D]), got {tuple(q.shape)}")
    q3 = q[:, 0] if q.dim() == 4 else q
    if q3.dim() != 3:
        raise ValueError(f"{where}: q must be [B, Hq, D] or [B, 1, Hq, D], got {tuple(q.shape)}")
    shape = q3.shape
    _ints(where, "cache_seqlens", cache_seqlens, shape[0])
    if softmax_scale is None:
        softmax_scale = shape[-1] ** -0.5
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _result(where, "out", out, q.shape, q.dtype)
        _apart(where, out, q)
    if lse is None:
        lse = q.new_empty(shape[:2], dtype=torch.float32)
    else:
        _result(where, "lse", lse, shape[:2], torch.float32)
    hq, d = shape[1:]
    ks, vs, pages, page, hkv, layout = _caches(where, q, d, k_cache, v_cache, kv_layout)
    if hq % hkv:
        raise ValueError(f"{where}: num_q_heads {hq} must be a multiple of num_kv_heads {hkv}")
    if q3.stride(2) != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    if k_scale is not None or v_scale is not None:
        _scales(where, hkv, k_scale, v_scale)
    _table(where, "block_table", block_table, shape[0])
    out3 = out[:, 0] if out.dim() == 4 else out
    fp8 = k_cache.dtype is torch.float8_e4m3fn
    qs, so = q3.stride(), out3.stride()
    a = _lib.SharedPrefixArgs((
        q3.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), *ks, *vs, pages,
        cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0),
        _ptr(k_scale) if fp8 else None, _ptr(v_scale) if fp8 else None,
        out3.data_ptr(), so[0], so[1], lse.data_ptr(), lse.stride(0),
        shape[0], hq, hkv, d, page, block_table.shape[1], _DT[q.dtype], _DT[k_cache.dtype],
        softmax_scale, None, 0, num_ctas or 0, flags, layout, wait_limit_us),
        prefix_lens.data_ptr(), prefix_block_table.data_ptr(), prefix_block_table.stride(0), _ptr(group_starts),
        groups, prefix_block_table.shape[1])
    own = a.own
    lib = _lib.load()
    with _on(index):
        _call(lib.b2d_decode_shared_prefix, "b2d_decode_shared_prefix", a, own, workspace, index,
              lib.b2d_shared_prefix_workspace_bytes)
    return out, lse


_MERGE = {torch.bfloat16: _lib.B2D_BF16, torch.float16: _lib.B2D_FP16, torch.float32: _lib.B2D_FP32}


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First and last byte address + 1 that a (non-empty) tensor covers."""
    first, elems = t.data_ptr(), 1
    if t.is_contiguous():
        return first, first + t.nbytes
    for n, s in zip(t.shape, t.stride()):
        elems += (n - 1) * s
    return first, first + elems * t.element_size()


def merge_states(outs: torch.Tensor, lses: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                 lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Merge attention states over disjoint parts of the keys into the state
    over all of them: out = sum_i e^(lse_i - M) out_i / sum_i e^(lse_i - M),
    lse = M + ln sum_i e^(lse_i - M), M = max_i lse_i.

    outs [N, T, H, D] (bf16, fp16 or fp32, D a multiple of 8 up to 1024) and lses
    [N, T, H] fp32 (natural log), e.g. the (out, lse) of decode() calls over
    parts of a cache, written into one buffer with out= and lse=, or gathered
    from context-parallel ranks.  A state with lse = -inf is not read; rows in
    which all are give out = 0, lse = -inf.  Returns out [T, H, D] in outs'
    dtype (fp32 states: in the dtype of a given `out`) and lse [T, H]; neither
    may overlap the inputs."""
    where = "merge_states"
    if not outs.is_cuda:
        raise RuntimeError("b200decode.merge_states needs CUDA tensors (there is no CPU path)")
    if outs.dim() != 4 or outs.dtype not in _MERGE:
        raise ValueError(f"{where}: outs must be bf16, fp16 or fp32 [N, T, H, D], got {outs.dtype} {tuple(outs.shape)}")
    shape = outs.shape
    if lses.dtype is not torch.float32 or lses.shape != shape[:3]:
        raise ValueError(f"{where}: lses must be fp32 {list(shape[:3])}")
    so, sl = outs.stride(), lses.stride()
    if so[3] != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    index = outs.get_device()
    _one_device(where, index, lses, out, lse)
    n, t, h, d = shape
    given = [x for x in (out, lse) if x is not None]
    if out is None:
        out = outs.new_empty((t, h, d))
    else:
        if (out.dtype is not outs.dtype and outs.dtype is not torch.float32) or out.dtype not in _MERGE:
            raise ValueError(f"{where}: out must be {outs.dtype} like the states, or 16-bit from fp32 states")
        _result(where, "out", out, shape[1:], out.dtype)
    if lse is None:
        lse = lses.new_empty((t, h))
    elif lse.dtype is not torch.float32 or lse.shape != shape[1:3]:
        raise ValueError(f"{where}: lse must be fp32 [{t}, {h}]")
    if given and out.numel():
        (o0, o1), (l0, l1) = _span(outs), _span(lses)
        for x in given:
            first, end = _span(x)
            if (first < o1 and o0 < end) or (first < l1 and l0 < end):
                raise ValueError(f"{where}: out or lse overlaps an input")
    wo, wl = out.stride(), lse.stride()
    a = _lib.MergeArgs(outs.data_ptr(), so[0], so[1], so[2], lses.data_ptr(), sl[0], sl[1], sl[2],
                       out.data_ptr(), wo[0], wo[1], lse.data_ptr(), wl[0], wl[1],
                       n, t, h, d, _MERGE[outs.dtype], _MERGE[out.dtype])
    with _on(index):
        rc = _lib.load().b2d_merge_states(C.byref(a), _stream(index))
    if rc:
        raise B2DError(rc, "b2d_merge_states")
    return out, lse
