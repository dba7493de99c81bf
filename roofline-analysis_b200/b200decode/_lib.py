"""ctypes binding of libb2d.so (include/b2d_decode.h).

The structures below mirror the header's argument structures field for field.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "_native" / "libb2d.so"

B2D_KV_STRIDED, B2D_KV_VLLM = 0, 1
B2D_BF16, B2D_FP16, B2D_FP8_E4M3, B2D_FP32 = 0, 1, 2, 3
B2D_FLAG_SKIP_COMBINE, B2D_FLAG_COMBINE_ONLY, B2D_FLAG_TEST_NO_LOADS = 1, 2, 4
B2D_WORKSPACE_HEADER_BYTES = 65792
B2D_ERR_UNSUPPORTED, B2D_ERR_WORKSPACE, B2D_ERR_DEVICE_CAPACITY = -2, -4, -9

EXPORTED = (
    "b2d_gqa_workspace_bytes",
    "b2d_decode_gqa",
    "b2d_decode_gqa_static_scratch",
    "b2d_mla_workspace_bytes",
    "b2d_decode_mla",
    "b2d_check_device_status",
    "b2d_append_kv",
    "b2d_gqa_plan",
    "b2d_cross_workspace_bytes",
    "b2d_cross_attention",
    "b2d_shared_prefix_workspace_bytes",
    "b2d_decode_shared_prefix",
    "b2d_merge_states",
    "b2d_plan_append",
    "b2d_release_pages",
    "b2d_error_string",
    "b2d_version",
)


class GqaArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("q_stride_b", C.c_int64), ("q_stride_h", C.c_int64),
        ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
        ("k_stride_page", C.c_int64), ("k_stride_tok", C.c_int64), ("k_stride_head", C.c_int64),
        ("v_stride_page", C.c_int64), ("v_stride_tok", C.c_int64), ("v_stride_head", C.c_int64),
        ("num_pages", C.c_int64),
        ("cache_seqlens", C.c_void_p), ("block_table", C.c_void_p),
        ("block_table_stride", C.c_int64),
        ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("out", C.c_void_p), ("out_stride_b", C.c_int64), ("out_stride_h", C.c_int64),
        ("lse", C.c_void_p), ("lse_stride_b", C.c_int64),
        ("batch", C.c_int32), ("num_q_heads", C.c_int32), ("num_kv_heads", C.c_int32),
        ("head_dim", C.c_int32), ("page_size", C.c_int32), ("max_pages_per_seq", C.c_int32),
        ("q_dtype", C.c_int32), ("kv_dtype", C.c_int32),
        ("softmax_scale", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("num_ctas", C.c_int32), ("flags", C.c_int32), ("kv_layout", C.c_int32),
        ("wait_limit_us", C.c_int32),
    ]


class MlaArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("q_stride_b", C.c_int64), ("q_stride_h", C.c_int64),
        ("kv_cache", C.c_void_p), ("kv_stride_page", C.c_int64), ("kv_stride_tok", C.c_int64),
        ("num_pages", C.c_int64),
        ("cache_seqlens", C.c_void_p), ("block_table", C.c_void_p),
        ("block_table_stride", C.c_int64),
        ("out", C.c_void_p), ("out_stride_b", C.c_int64), ("out_stride_h", C.c_int64),
        ("lse", C.c_void_p), ("lse_stride_b", C.c_int64),
        ("batch", C.c_int32), ("num_heads", C.c_int32), ("head_dim_qk", C.c_int32),
        ("head_dim_v", C.c_int32), ("page_size", C.c_int32), ("max_pages_per_seq", C.c_int32),
        ("dtype", C.c_int32), ("softmax_scale", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("num_ctas", C.c_int32), ("flags", C.c_int32), ("wait_limit_us", C.c_int32),
        ("reserved", C.c_int32),
    ]


class AppendArgs(C.Structure):
    _fields_ = [
        ("key", C.c_void_p), ("value", C.c_void_p),
        ("src_stride_t", C.c_int64), ("src_stride_h", C.c_int64),
        ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
        ("k_stride_page", C.c_int64), ("k_stride_tok", C.c_int64), ("k_stride_head", C.c_int64),
        ("v_stride_page", C.c_int64), ("v_stride_tok", C.c_int64), ("v_stride_head", C.c_int64),
        ("num_pages", C.c_int64), ("slot_mapping", C.c_void_p),
        ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("bad_slots", C.c_void_p),
        ("num_tokens", C.c_int32), ("num_kv_heads", C.c_int32), ("head_dim", C.c_int32),
        ("page_size", C.c_int32), ("src_dtype", C.c_int32), ("cache_dtype", C.c_int32),
        ("kv_layout", C.c_int32), ("reserved", C.c_int32),
    ]


class CrossArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("q_stride_t", C.c_int64), ("q_stride_h", C.c_int64),
        ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
        ("k_stride_page", C.c_int64), ("k_stride_tok", C.c_int64), ("k_stride_head", C.c_int64),
        ("v_stride_page", C.c_int64), ("v_stride_tok", C.c_int64), ("v_stride_head", C.c_int64),
        ("num_pages", C.c_int64),
        ("query_starts", C.c_void_p), ("kv_lens", C.c_void_p), ("block_table", C.c_void_p),
        ("block_table_stride", C.c_int64),
        ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("out", C.c_void_p), ("out_stride_t", C.c_int64), ("out_stride_h", C.c_int64),
        ("lse", C.c_void_p), ("lse_stride_t", C.c_int64),
        ("num_tokens", C.c_int32), ("num_groups", C.c_int32), ("query_len", C.c_int32),
        ("num_q_heads", C.c_int32), ("num_kv_heads", C.c_int32), ("head_dim", C.c_int32),
        ("page_size", C.c_int32), ("max_pages_per_seq", C.c_int32),
        ("q_dtype", C.c_int32), ("kv_dtype", C.c_int32), ("softmax_scale", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("num_ctas", C.c_int32), ("flags", C.c_int32), ("kv_layout", C.c_int32),
        ("wait_limit_us", C.c_int32),
    ]


class SharedPrefixArgs(C.Structure):
    _fields_ = [
        ("own", GqaArgs),
        ("prefix_lens", C.c_void_p), ("prefix_block_table", C.c_void_p),
        ("prefix_block_table_stride", C.c_int64), ("group_starts", C.c_void_p),
        ("num_groups", C.c_int32), ("prefix_max_pages", C.c_int32),
    ]


class MergeArgs(C.Structure):
    _fields_ = [
        ("outs", C.c_void_p), ("outs_stride_n", C.c_int64), ("outs_stride_t", C.c_int64),
        ("outs_stride_h", C.c_int64),
        ("lses", C.c_void_p), ("lses_stride_n", C.c_int64), ("lses_stride_t", C.c_int64),
        ("lses_stride_h", C.c_int64),
        ("out", C.c_void_p), ("out_stride_t", C.c_int64), ("out_stride_h", C.c_int64),
        ("lse", C.c_void_p), ("lse_stride_t", C.c_int64), ("lse_stride_h", C.c_int64),
        ("num_states", C.c_int32), ("num_tokens", C.c_int32), ("num_heads", C.c_int32),
        ("head_dim", C.c_int32), ("in_dtype", C.c_int32), ("out_dtype", C.c_int32),
    ]


class PlanAppendArgs(C.Structure):
    _fields_ = [
        ("cache_seqlens", C.c_void_p), ("new_tokens", C.c_void_p), ("block_table", C.c_void_p),
        ("block_table_stride", C.c_int64), ("free_pages", C.c_void_p), ("free_count", C.c_void_p),
        ("slot_mapping", C.c_void_p), ("query_starts", C.c_void_p), ("seqlens_out", C.c_void_p),
        ("free_count_out", C.c_void_p),
        ("num_requests", C.c_int32), ("max_pages_per_seq", C.c_int32), ("page_size", C.c_int32),
        ("max_tokens", C.c_int32), ("free_capacity", C.c_int32), ("reserved", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class ReleaseArgs(C.Structure):
    _fields_ = [
        ("cache_seqlens", C.c_void_p), ("finished", C.c_void_p), ("block_table", C.c_void_p),
        ("block_table_stride", C.c_int64), ("free_pages", C.c_void_p), ("free_count", C.c_void_p),
        ("seqlens_out", C.c_void_p), ("free_count_out", C.c_void_p),
        ("num_requests", C.c_int32), ("max_pages_per_seq", C.c_int32), ("page_size", C.c_int32),
        ("free_capacity", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


_lib = None


def load() -> C.CDLL:
    """Load libb2d.so once; raise (never fall back) when it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    path = Path(os.environ.get("B2D_LIBRARY", LIB_PATH))
    if not path.exists():
        raise RuntimeError(
            f"libb2d.so not found at {path}; build it with "
            "`python roofline-analysis_b200/build.py` (there is no CPU fallback)")
    lib = C.CDLL(str(path))
    lib.b2d_gqa_workspace_bytes.argtypes = [C.POINTER(GqaArgs), C.POINTER(C.c_size_t)]
    lib.b2d_decode_gqa.argtypes = [C.POINTER(GqaArgs), C.c_void_p]
    lib.b2d_decode_gqa_static_scratch.argtypes = [C.POINTER(GqaArgs), C.c_void_p]
    lib.b2d_mla_workspace_bytes.argtypes = [C.POINTER(MlaArgs), C.POINTER(C.c_size_t)]
    lib.b2d_decode_mla.argtypes = [C.POINTER(MlaArgs), C.c_void_p]
    lib.b2d_append_kv.argtypes = [C.POINTER(AppendArgs), C.c_void_p]
    lib.b2d_check_device_status.argtypes = [C.c_void_p, C.c_int, C.c_void_p]
    lib.b2d_static_scratch_check_status.argtypes = [C.c_int, C.c_void_p]
    lib.b2d_gqa_launch_count.argtypes = [C.POINTER(GqaArgs), C.POINTER(C.c_int32)]
    lib.b2d_cross_workspace_bytes.argtypes = [C.POINTER(CrossArgs), C.POINTER(C.c_size_t)]
    lib.b2d_cross_attention.argtypes = [C.POINTER(CrossArgs), C.c_void_p]
    lib.b2d_shared_prefix_workspace_bytes.argtypes = [C.POINTER(SharedPrefixArgs),
                                                      C.POINTER(C.c_size_t)]
    lib.b2d_decode_shared_prefix.argtypes = [C.POINTER(SharedPrefixArgs), C.c_void_p]
    lib.b2d_merge_states.argtypes = [C.POINTER(MergeArgs), C.c_void_p]
    lib.b2d_plan_append.argtypes = [C.POINTER(PlanAppendArgs), C.c_void_p]
    lib.b2d_release_pages.argtypes = [C.POINTER(ReleaseArgs), C.c_void_p]
    lib.b2d_gqa_plan.argtypes = [C.POINTER(GqaArgs), C.POINTER(C.c_int32), C.POINTER(C.c_int32),
                                 C.POINTER(C.c_int32)]
    lib.b2d_error_string.restype = C.c_char_p
    lib.b2d_error_string.argtypes = [C.c_int]
    lib.b2d_version.restype = C.c_char_p
    _lib = lib
    return lib
