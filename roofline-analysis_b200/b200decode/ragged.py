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

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from .api import _DT, DecodeWorkspace, _check, _default_ws, _gqa_args, _layout_strides, _ptr, decode


def _one_device(where: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{where}: {name} is on {t.device}, q on {device}")


def _ints(where: str, shape: tuple, **tensors) -> None:
    for name, t in tensors.items():
        if t.dtype != torch.int32 or tuple(t.shape) != shape:
            raise ValueError(f"{where}: {name} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{where}: {name} must be contiguous")


def _result(where: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.stride(-1) != 1:
        raise ValueError(f"{where}: {name} must be {dtype} {list(shape)} with a contiguous last axis")


def _workspace(workspace: Optional[DecodeWorkspace], device: torch.device, need: int) -> DecodeWorkspace:
    """The caller's workspace, or the default one of the device's current
    stream.  While that stream is captured into a CUDA graph the default would
    be shared by every graph captured there, and could be reallocated under
    them: a call without a workspace of its own then gets one from the graph's
    memory pool (its header is zeroed by a node of the graph)."""
    capturing = torch.cuda.is_current_stream_capturing()
    if workspace is not None:
        if workspace.buf.device != device:
            raise ValueError(f"workspace is on {workspace.buf.device}, the tensors on {device}")
        workspace.captured = workspace.captured or capturing
        return workspace.ensure(need)
    if capturing:
        return DecodeWorkspace.in_graph(device, need)
    return _default_ws(device).ensure(need)


def _cache_fields(a: _lib.CrossArgs, where: str, q: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, kv_layout: str) -> int:
    """Fills the cache fields of `a`; returns the number of KV heads."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{where}: q dtype must be bf16 or fp16, got {q.dtype}")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (q.dtype, torch.float8_e4m3fn):
        raise ValueError(f"{where}: cache dtype {k_cache.dtype} must equal q's {q.dtype} or be float8_e4m3fn")
    d = q.shape[-1]
    if kv_layout == "vllm":
        if k_cache.dim() != 5 or v_cache.dim() != 4 or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError(f"{where}: kv_layout='vllm' takes contiguous K [blocks, Hkv, D/x, P, x] and V "
                             "[blocks, Hkv, D, P]")
        nb, hkv, dx, page, x = k_cache.shape
        if x * k_cache.element_size() != 16 or tuple(v_cache.shape) != (nb, hkv, dx * x, page) or dx * x != d:
            raise ValueError(f"{where}: vLLM cache shapes do not match")
        ks, vs = (k_cache.stride(0), x, k_cache.stride(1)), (v_cache.stride(0), 1, v_cache.stride(1))
        a.kv_layout = _lib.B2D_KV_VLLM
    else:
        if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
            raise ValueError(f"{where}: k_cache and v_cache must be matching 4-D paged caches")
        if k_cache.stride(-1) != 1 or v_cache.stride(-1) != 1:
            raise ValueError(f"{where}: the head_dim axis must be contiguous")
        if k_cache.shape[-1] != d:
            raise ValueError(f"{where}: head_dim mismatch between q and the caches")
        *ks, page, hkv = _layout_strides(k_cache, kv_layout)
        *vs, _, _ = _layout_strides(v_cache, kv_layout)
        a.kv_layout = _lib.B2D_KV_STRIDED
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.k_stride_page, a.k_stride_tok, a.k_stride_head = ks
    a.v_stride_page, a.v_stride_tok, a.v_stride_head = vs
    a.num_pages, a.page_size, a.num_kv_heads = k_cache.shape[0], page, hkv
    return hkv


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
    kernel.  Caches, scales and layouts as in decode(); kv_lens int32 [B],
    block_table int32 [B, max_pages].  softmax_scale defaults to 1/sqrt(D).
    Returns out (shape of q) and lse (shape of q without D, fp32, natural
    log).  A request without states gives out = 0, lse = -inf; ragged tokens
    behind query_starts[B] are left as they were.

    Captured into a CUDA graph without `workspace`, a call keeps its scratch
    in the graph's memory pool; check_device_status() reads the status only of
    a workspace that the caller passes.
    """
    where = "cross_attention"
    if not q.is_cuda:
        raise RuntimeError("b200decode.cross_attention needs CUDA tensors (there is no CPU path)")
    ragged = query_starts is not None
    if q.dim() != (3 if ragged else q.dim()) or q.dim() not in (3, 4):
        raise ValueError(f"{where}: q must be [T, Hq, D] with query_starts, or [B, Tq, Hq, D] or [B, Hq, D] "
                         f"without, got {tuple(q.shape)}")
    bsz = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    _ints(where, (bsz,), kv_lens=kv_lens)
    _one_device(where, q.device, k_cache=k_cache, v_cache=v_cache, kv_lens=kv_lens, block_table=block_table,
                query_starts=query_starts, k_scale=k_scale, v_scale=v_scale, out=out, lse=lse)
    if not ragged and q.shape[0] != bsz:
        raise ValueError(f"{where}: q has {q.shape[0]} requests, kv_lens {bsz}")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != bsz:
        raise ValueError(f"{where}: block_table must be int32 [{bsz}, max_pages]")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError(f"{where}: block_table rows must be contiguous")
    if q.stride(-1) != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
    _result(where, "out", out, q.shape, q.dtype)
    _result(where, "lse", lse, q.shape[:-1], torch.float32)
    a = _lib.CrossArgs()
    hkv = _cache_fields(a, where, q, k_cache, v_cache, kv_layout)
    hq, d = q.shape[-2:]
    if hq % hkv:
        raise ValueError(f"{where}: num_q_heads {hq} must be a multiple of num_kv_heads {hkv}")
    for s, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if s is not None and (s.dtype != torch.float32 or s.numel() != hkv or not s.is_contiguous()):
            raise ValueError(f"{where}: {n} must be contiguous fp32 with num_kv_heads elements")
    if ragged:
        _ints(where, (bsz + 1,), query_starts=query_starts)
        q3, out3, lse2, length = q, out, lse, 0
    elif q.dim() == 4:
        # [B, Tq, ...] as [B * Tq, ...]: one token stride
        q3 = q.reshape(-1, hq, d)
        try:
            out3, lse2 = out.view(-1, hq, d), lse.view(-1, hq)
        except RuntimeError as e:
            raise ValueError(f"{where}: out and lse need one stride for all tokens") from e
        length = q.shape[1]
    else:
        q3, out3, lse2, length = q, out, lse, 1
    if q3.shape[0] == 0 or bsz == 0:
        return out, lse
    with torch.cuda.device(q.device):
        if length == 1 and not flags:
            ws = workspace
            if ws is not None or torch.cuda.is_current_stream_capturing():
                g = _gqa_args(q3, k_cache, v_cache, kv_lens, block_table, softmax_scale, k_scale, v_scale, out3,
                              lse2, kv_layout, num_ctas)
                need = C.c_size_t(0)
                _check(_lib.load().b2d_gqa_workspace_bytes(C.byref(g), C.byref(need)), "b2d_gqa_workspace_bytes")
                ws = _workspace(workspace, q.device, need.value)
            decode(q3, k_cache, v_cache, kv_lens, block_table, softmax_scale, k_scale=k_scale, v_scale=v_scale,
                   out=out3, lse=lse2, kv_layout=kv_layout, num_ctas=num_ctas, workspace=ws,
                   wait_limit_us=wait_limit_us)
            return out, lse
        a.q, a.q_stride_t, a.q_stride_h = q3.data_ptr(), q3.stride(0), q3.stride(1)
        a.query_starts, a.kv_lens, a.block_table = _ptr(query_starts), kv_lens.data_ptr(), block_table.data_ptr()
        a.block_table_stride = block_table.stride(0)
        fp8 = k_cache.dtype == torch.float8_e4m3fn
        a.k_scale, a.v_scale = (_ptr(k_scale), _ptr(v_scale)) if fp8 else (None, None)
        a.out, a.out_stride_t, a.out_stride_h = out3.data_ptr(), out3.stride(0), out3.stride(1)
        a.lse, a.lse_stride_t = lse2.data_ptr(), lse2.stride(0)
        a.num_tokens, a.num_groups, a.query_len = q3.shape[0], bsz, length
        a.num_q_heads, a.head_dim, a.max_pages_per_seq = hq, d, block_table.shape[1]
        a.q_dtype, a.kv_dtype = _DT[q.dtype], _DT[k_cache.dtype]
        a.softmax_scale, a.num_ctas = float(softmax_scale), int(num_ctas or 0)
        a.flags, a.wait_limit_us = int(flags), int(wait_limit_us)
        lib = _lib.load()
        need = C.c_size_t(0)
        _check(lib.b2d_cross_workspace_bytes(C.byref(a), C.byref(need)), "b2d_cross_workspace_bytes")
        ws = _workspace(workspace, q.device, need.value)
        a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
        _check(lib.b2d_cross_attention(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)),
               "b2d_cross_attention")
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
    outside every group have no prefix); None: one group with the whole batch.
    The rest as in decode().  Out is computed in fp32 over both parts and
    rounded once.

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
    _one_device(where, q.device, k_cache=k_cache, v_cache=v_cache, prefix_lens=prefix_lens,
                prefix_block_table=prefix_block_table, cache_seqlens=cache_seqlens, block_table=block_table,
                group_starts=group_starts, k_scale=k_scale, v_scale=v_scale, out=out, lse=lse)
    groups = prefix_lens.shape[0] if prefix_lens.dim() == 1 else -1
    _ints(where, (groups,), prefix_lens=prefix_lens)
    if group_starts is not None:
        _ints(where, (groups + 1,), group_starts=group_starts)
    elif groups > 1:
        raise ValueError(f"{where}: {groups} prefixes need group_starts")
    if (prefix_block_table.dtype != torch.int32 or prefix_block_table.dim() != 2
            or prefix_block_table.shape[0] != groups):
        raise ValueError(f"{where}: prefix_block_table must be int32 [{groups}, max_pages]")
    if prefix_block_table.stride(1) != 1 and prefix_block_table.shape[1] > 1:
        raise ValueError(f"{where}: prefix_block_table rows must be contiguous")
    q3 = q[:, 0] if q.dim() == 4 else q
    if q3.dim() != 3:
        raise ValueError(f"{where}: q must be [B, Hq, D] or [B, 1, Hq, D], got {tuple(q.shape)}")
    if not cache_seqlens.is_contiguous():
        raise ValueError(f"{where}: cache_seqlens must be contiguous")
    for s, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if s is not None and not s.is_contiguous():
            raise ValueError(f"{where}: {n} must be contiguous")
    if softmax_scale is None:
        softmax_scale = q3.shape[-1] ** -0.5
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty(q3.shape[:2], dtype=torch.float32, device=q.device)
    _result(where, "out", out, q.shape, q.dtype)
    _result(where, "lse", lse, q3.shape[:2], torch.float32)
    out3 = out[:, 0] if out.dim() == 4 else out
    with torch.cuda.device(q.device):
        a = _lib.SharedPrefixArgs()
        a.own = _gqa_args(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, k_scale, v_scale,
                          out3, lse, kv_layout, num_ctas)
        a.own.flags, a.own.wait_limit_us = int(flags), int(wait_limit_us)
        a.prefix_lens, a.prefix_block_table = prefix_lens.data_ptr(), prefix_block_table.data_ptr()
        a.prefix_block_table_stride = prefix_block_table.stride(0)
        a.group_starts = _ptr(group_starts)
        a.num_groups, a.prefix_max_pages = groups, prefix_block_table.shape[1]
        lib = _lib.load()
        need = C.c_size_t(0)
        _check(lib.b2d_shared_prefix_workspace_bytes(C.byref(a), C.byref(need)),
               "b2d_shared_prefix_workspace_bytes")
        ws = _workspace(workspace, q.device, need.value)
        a.own.workspace, a.own.workspace_bytes = ws.ptr, ws.nbytes
        _check(lib.b2d_decode_shared_prefix(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)),
               "b2d_decode_shared_prefix")
    return out, lse


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First and last byte address + 1 that a (non-empty) tensor covers."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


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
    if outs.dim() != 4 or outs.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{where}: outs must be bf16, fp16 or fp32 [N, T, H, D], got {outs.dtype} {tuple(outs.shape)}")
    if lses.dtype != torch.float32 or lses.shape != outs.shape[:3]:
        raise ValueError(f"{where}: lses must be fp32 {list(outs.shape[:3])}")
    if outs.stride(3) != 1:
        raise ValueError(f"{where}: the head_dim axis must be contiguous")
    _one_device(where, outs.device, lses=lses, out=out, lse=lse)
    n, t, h, d = outs.shape
    if out is None:
        out = torch.empty(t, h, d, dtype=outs.dtype, device=outs.device)
    if lse is None:
        lse = torch.empty(t, h, dtype=torch.float32, device=outs.device)
    if out.dtype != outs.dtype and outs.dtype != torch.float32:
        raise ValueError(f"{where}: out must be {outs.dtype} like the states")
    if out.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{where}: out must be bf16, fp16 or fp32, got {out.dtype}")
    _result(where, "out", out, (t, h, d), out.dtype)
    if lse.dtype != torch.float32 or tuple(lse.shape) != (t, h):
        raise ValueError(f"{where}: lse must be fp32 [{t}, {h}]")
    if out.numel():
        spans = [(_span(x), f"{name}") for x, name in ((outs, "outs"), (lses, "lses"))]
        for x, name in ((out, "out"), (lse, "lse")):
            a0, a1 = _span(x)
            for (b0, b1), other in spans:
                if a0 < b1 and b0 < a1:
                    raise ValueError(f"{where}: {name} overlaps {other}")
    a = _lib.MergeArgs()
    a.outs, a.outs_stride_n, a.outs_stride_t, a.outs_stride_h = outs.data_ptr(), *outs.stride()[:3]
    a.lses, a.lses_stride_n, a.lses_stride_t, a.lses_stride_h = lses.data_ptr(), *lses.stride()
    a.out, a.out_stride_t, a.out_stride_h = out.data_ptr(), *out.stride()[:2]
    a.lse, a.lse_stride_t, a.lse_stride_h = lse.data_ptr(), *lse.stride()
    a.num_states, a.num_tokens, a.num_heads, a.head_dim = n, t, h, d
    dt = {**_DT, torch.float32: _lib.B2D_FP32}
    a.in_dtype, a.out_dtype = dt[outs.dtype], dt[out.dtype]
    with torch.cuda.device(outs.device):
        _check(_lib.load().b2d_merge_states(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)),
               "b2d_merge_states")
    return out, lse
