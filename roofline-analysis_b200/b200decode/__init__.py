"""b200decode — B200-native (sm_100a) paged decode attention.

Host layer over libb2d.so (hand-written CUDA kernels behind a C ABI,
include/b2d_decode.h).  Public API:

    decode(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale)
        -> (out, lse)
    decode_mla(q, kv_cache, cache_seqlens, block_table, softmax_scale)
        -> (out, lse)
    append_kv(key, value, k_cache, v_cache, slot_mapping)     (reshape_and_cache)
    decode_shared_prefix(q, k_cache, v_cache, prefix_lens, prefix_block_table,
        cache_seqlens, block_table, ...) -> (out, lse)        (prefixes read once per group)
    cross_attention(q, k_cache, v_cache, kv_lens, block_table, ...) -> (out, lse)
        (ragged query tokens over paged encoder states)
    merge_states(outs, lses) -> (out, lse)                    (states over disjoint keys)
    plan_append(cache_seqlens, block_table, free_pages, free_count, page_size, ...)
        -> AppendPlan; release_pages(...)                     (block tables on the GPU)
    GqaDecoder(...).run() / .capture() / .replay()           (plan once, CUDA graphs)
    cluster_decode.cluster_decode_forward(q, k, v, config)   (the reference's own
        dense decode entry point)
    python -m b200decode.decodebench [mla] ...               (decodebench backend)

There is no CPU or library fallback: calling either without the compiled
library or without a CUDA device raises.
"""
from .api import (  # noqa: F401
    B2DError,
    append_kv,
    DecodeWorkspace,
    GqaDecoder,
    check_device_status,
    decode,
    decode_mla,
    gqa_plan,
    library_path,
)

from .pages import AppendPlan, plan_append, release_pages  # noqa: F401,E402
from .ragged import cross_attention, decode_shared_prefix, merge_states  # noqa: F401,E402
from . import cluster_decode  # noqa: F401,E402

__version__ = "0.1.0"
