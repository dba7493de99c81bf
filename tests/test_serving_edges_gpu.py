"""Serving operators where they can go wrong: pages that a pool must not get,
sizes that one path takes and another does not, rows without mass, weights far
below the largest, and errors that a bound for each element does not see."""
import threading

import pytest
import torch

import b200decode
from b200decode import _lib
from serving_ref import attend, caches, check, check_lse, gather, merge2, tables, u_of

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def i32(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def paged(device, seed, lens, P, hkv, d, kv, layout="NHD"):
    """Caches with sequences `lens` in them, pages in random order."""
    gen = torch.Generator(device=device).manual_seed(seed)
    pages = sum((n + P - 1) // P for n in lens) + 2
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    k, v, ks, vs = caches(gen, device, pages, P, hkv, d, kv, layout)
    return gen, k, v, ks, vs, tables(lens, P, perm, 0)[0].to(device)


def lay(layout, which):
    return f"vllm_{which}" if layout == "vllm" else layout



# ---------------------------------------------------------------- tiles

@pytest.mark.parametrize("hkv,grp,P", [(1, 2, 5), (3, 4, 5), (1, 16, 1), (5, 1, 7), (1, 4, 25), (3, 2, 3)])
@pytest.mark.parametrize("num_ctas", [None, 2])
def test_e4m3_tiles_of_any_number_of_bytes(cuda, hkv, grp, P, num_ctas):
    """e4m3 at head_dim 64 with an odd number of heads in a tile and an odd page:
    K and V tiles of 64 n bytes, n odd, each of which starts on its own 128-byte
    boundary in shared memory."""
    lens, plen = [1, 300, 0, 77], 130
    gen, k, v, ks, vs, both = paged(cuda, 290, lens + [plen], P, hkv, 64, F8)
    bt, pbt = both[:4], both[4:]
    q = torch.randn(4, hkv * grp, 64, generator=gen, device=cuda).to(BF)
    kw = dict(k_scale=ks, v_scale=vs, num_ctas=num_ctas)
    got = [b200decode.decode(q, k, v, i32(lens), bt, **kw),
           b200decode.decode_shared_prefix(q, k, v, i32([plen]), pbt, i32(lens), bt, **kw)]
    torch.cuda.synchronize()
    b200decode.check_device_status()
    for b, n in enumerate(lens):
        part = [attend(q[b:b + 1].double(), gather(k, ks, r, m, "NHD"), gather(v, vs, r, m, "NHD"), 0.125, F8)
                for r, m in ((bt[b], n), (pbt[0], plen))]
        for (out, lse), ref in zip(got, (part[0], merge2(*part))):
            check(out[b:b + 1], ref[0], ref[2], u_of(BF), "out")
            check_lse(lse[b:b + 1], ref[1], ref[3])
