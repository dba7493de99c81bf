"""Which sizes the serving calls take, asked on the host (no GPU needed)."""
import ctypes as C

import pytest

from b200decode import _lib

BF, HF, F8 = _lib.B2D_BF16, _lib.B2D_FP16, _lib.B2D_FP8_E4M3


def sizes(a, group, d, page, kv):
    a.num_kv_heads, a.num_q_heads, a.head_dim, a.page_size = 2, 2 * group, d, page
    a.max_pages_per_seq, a.num_ctas = 64, 148
    a.q_dtype, a.kv_dtype = (HF if kv == HF else BF), kv
    return a


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("kv", [BF, HF, F8])
def test_cross_takes_every_group_and_shared_prefix_what_decode_takes(d, page, kv):
    lib, n = _lib.load(), C.c_size_t(0)
    refused = []
    for group in range(1, 33):
        c = sizes(_lib.CrossArgs(), group, d, page, kv)
        c.num_tokens, c.num_groups, c.query_len = 4, 4, 1
        assert lib.b2d_cross_workspace_bytes(C.byref(c), C.byref(n)) == 0, group
        s = _lib.SharedPrefixArgs()
        sizes(s.own, group, d, page, kv)
        s.own.batch, s.num_groups, s.prefix_max_pages = 4, 1, 10
        decode = lib.b2d_gqa_workspace_bytes(C.byref(s.own), C.byref(n))
        assert decode in (0, _lib.B2D_ERR_UNSUPPORTED)
        assert lib.b2d_shared_prefix_workspace_bytes(C.byref(s), C.byref(n)) == decode
        if decode:
            refused.append(group)
    if d == 192 and (page % 16 or kv == F8):
        assert refused == list(range(1, 33))
    elif page % 16 == 0 and not (kv == F8 and d == 64):
        # up to 8 equal parts of up to 16 query heads (8 at head_dim 192 and 256)
        most = 16 if d < 192 else 8
        assert refused == [g for g in range(1, 33) if not any(g % w == 0 and g // w <= most for w in range(1, 9))]
    else:
        assert refused == [g for g in range(1, 33) if g > (8 if g % 2 else 16)]


@pytest.mark.parametrize("kv_heads", [1, 4, 6, 7, 8, 16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("kv", [BF, F8])
def test_two_stages_of_a_tile_fit_an_sm(kv_heads, d, kv):
    """K and V tiles of 16 tokens, two stages of each, in 227 KB of shared memory,
    for tables of any width (short ones have narrower tiles)."""
    if kv == F8 and d == 192:
        return
    lib, a = _lib.load(), _lib.GqaArgs()
    ctas, tokens, heads = C.c_int32(), C.c_int32(), C.c_int32()
    for columns in (1, 100, 1 << 16):
        sizes(a, 4, d, 16, kv)
        a.batch, a.num_kv_heads, a.num_q_heads, a.max_pages_per_seq = 64, kv_heads, 4 * kv_heads, columns
        assert lib.b2d_gqa_plan(C.byref(a), C.byref(ctas), C.byref(tokens), C.byref(heads)) == 0
        assert kv_heads % heads.value == 0
        # beside the tiles: barriers, up to 2049 row starts, scan and alignment
        assert 4 * tokens.value * heads.value * d * (1 if kv == F8 else 2) <= 227 * 1024 - 10 * 1024
