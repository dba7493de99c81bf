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


# ---------------------------------------------------------------- pages

@pytest.mark.parametrize("B", [3, 900])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_of_a_negative_page_changes_nothing(cuda, B, in_place):
    """A negative entry among the pages of a finished request never enters the
    pool: the step is reported and changes no length, count or free page."""
    P, width = 16, 7
    bt = torch.arange(B * width, dtype=torch.int32, device=cuda).reshape(B, width)
    lens = torch.full((B,), 100, dtype=torch.int32, device=cuda)      # all 7 pages
    lens[1] = 33                                                      # 3 pages
    bt[1, 3] = -8                                                     # (not one of them)
    fin = torch.ones(B, dtype=torch.bool, device=cuda)
    fin[0] = False
    bt[0, 2] = -1                                                     # (not finished)
    free = torch.full((B * width + 5,), -5, dtype=torch.int32, device=cuda)
    free[:5] = i32([B * width + x for x in range(5)])
    ws = b200decode.DecodeWorkspace(cuda)
    for bad in (True, False):
        table, sl, fr, cnt = bt.clone(), lens.clone(), free.clone(), i32([5])
        if bad:
            table[B - 1, 4] = -3
        kw = dict(seqlens_out=sl, free_count_out=cnt) if in_place else {}
        after, count = b200decode.release_pages(sl, table, fin, fr, cnt, P, workspace=ws, **kw)
        torch.cuda.synchronize()
        if bad:
            with pytest.raises(b200decode.B2DError) as e:
                b200decode.check_device_status(ws)
            assert e.value.code == -7
            assert torch.equal(after, lens) and int(count) == 5
            assert torch.equal(fr[:5], free[:5])
        else:
            b200decode.check_device_status(ws)
            given = [int(x) for b in range(1, B) for x in table[b, :3 if b == 1 else 7].tolist()]
            assert int(count) == 5 + len(given) and fr[:int(count)].tolist() == free[:5].tolist() + given
            assert after.tolist() == [100] + [0] * (B - 1)


def test_release_of_a_length_beyond_the_table_changes_nothing(cuda):
    bt = torch.arange(8, dtype=torch.int32, device=cuda).reshape(2, 4)
    sl, free, cnt = i32([64, 65]), torch.zeros(8, dtype=torch.int32, device=cuda), i32([0])
    ws = b200decode.DecodeWorkspace(cuda)
    after, count = b200decode.release_pages(sl, bt, torch.tensor([True, True], device=cuda), free, cnt, 16, workspace=ws)
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -9
    assert after.tolist() == [64, 65] and int(count) == 0 and (free == 0).all()
    after, count = b200decode.release_pages(sl, bt, torch.tensor([True, False], device=cuda), free, cnt, 16, workspace=ws)
    b200decode.check_device_status(ws)
    assert after.tolist() == [0, 65] and free[:4].tolist() == [0, 1, 2, 3] and int(count) == 4


def test_plan_append_reports_a_negative_page_of_the_pool(cuda):
    free = i32([4, -6, 5])
    ws = b200decode.DecodeWorkspace(cuda)
    bt = torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    plan = b200decode.plan_append(i32([0, 0]), bt, free, i32([3]), 16, workspace=ws)
    assert plan.slot_mapping.tolist() == [80, -1]
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -7
    b200decode.plan_append(i32([0]), bt[:1], free, i32([3]), 16, workspace=ws)
    b200decode.check_device_status(ws)


# ---------------------------------------------------------------- two calls at once

def test_first_call_of_a_host_thread(cuda):
    """A thread whose first CUDA call is one of these, on tensors that another
    thread made."""
    lens = [40, 300]
    gen, k, v, _, _, bt = paged(cuda, 345, lens, 16, 2, 128, BF)
    q, kl, st = torch.randn(2, 8, 128, generator=gen, device=cuda).to(BF), i32(lens), i32([0, 1, 2])
    out, lse = torch.empty_like(q), torch.empty(2, 8, device=cuda)
    calls = [lambda: b200decode.decode(q, k, v, kl, bt, out=out, lse=lse),
             lambda: b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, out=out, lse=lse),
             lambda: b200decode.cross_attention(q, k, v, kl, bt, out=out, lse=lse),
             lambda: b200decode.decode_shared_prefix(q, k, v, kl[:1], bt[:1], kl, bt, out=out, lse=lse)]
    for call in calls:
        want = [x.clone() for x in call()]
        torch.cuda.synchronize()
        got = []

        def work():
            try:
                got.extend(x.clone() for x in call())
            except Exception as e:   # noqa: BLE001
                got.append(e)

        t = threading.Thread(target=work)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert len(got) == 2, got
        assert all(torch.equal(x, y) for x, y in zip(got, want))

def test_host_threads_on_one_stream(cuda):
    """Threads that share a stream share its default workspace: the launches of
    one call are not mixed with another's."""
    P, hkv, hq, d = 16, 2, 8, 128
    lens = [900, 700, 300, 40, 500]
    gen, k, v, _, _, bt = paged(cuda, 350, lens, P, hkv, d, BF)
    kl = i32(lens)
    qs = [torch.randn(40, hq, d, generator=gen, device=cuda).to(BF) for _ in range(4)]
    own, obt = i32([300 + i for i in range(40)]), bt[1:2].repeat(40, 1)
    pool = torch.arange(1000, dtype=torch.int32, device=cuda)
    calls = [
        lambda: b200decode.decode_shared_prefix(qs[0], k, v, kl[:1], bt[:1], own, obt),
        lambda: b200decode.decode_shared_prefix(qs[1], k, v, kl[2:3], bt[2:3], own, obt, softmax_scale=0.2),
        lambda: b200decode.cross_attention(qs[2], k, v, kl, bt, query_starts=i32([0, 9, 20, 21, 30, 40])),
        lambda: b200decode.decode(qs[3][:5], k, v, kl, bt),
        lambda: b200decode.plan_append(kl, bt.clone(), pool, i32([1000]), P)[:3],
    ]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    wrong, ready = [], threading.Barrier(len(calls))

    def work(i):
        try:
            ready.wait()
            got = [calls[i]() for _ in range(60)]
            torch.cuda.synchronize()
            for g in got:
                if not all(torch.equal(x, y) for x, y in zip(g, want[i])):
                    wrong.append(i)
        except Exception as e:   # noqa: BLE001
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    b200decode.check_device_status()


# ---------------------------------------------------------------- sizes

ONE_TOKEN = [
    # Hq, Hkv, D, P, q dtype, cache dtype: sizes that decode()'s kernels do not take, and two that they do
    (9, 1, 128, 5, BF, BF), (32, 1, 128, 8, BF, BF), (11, 1, 256, 16, BF, BF), (17, 1, 128, 16, HF, HF),
    (62, 2, 128, 16, BF, BF), (32, 1, 64, 16, BF, F8), (11, 1, 64, 16, HF, F8), (26, 1, 256, 16, BF, F8),
    (8, 2, 192, 5, BF, BF), (8, 2, 192, 16, HF, F8), (16, 1, 128, 16, BF, BF), (8, 2, 192, 16, BF, BF),
]


@pytest.mark.parametrize("case", range(len(ONE_TOKEN)))
@pytest.mark.parametrize("form", ["BHD", "B1HD", "workspace", "captured"])
def test_cross_attention_of_one_token_takes_every_group(cuda, case, form):
    """Up to 32 query heads per KV head at every head_dim, page size and cache
    type, as with several tokens."""
    hq, hkv, d, P, qd, kv = ONE_TOKEN[case]
    lens = [1, 300, 0, 77]
    gen, k, v, ks, vs, bt = paged(cuda, 300 + case, lens, P, hkv, d, kv)
    q = torch.randn(4, hq, d, generator=gen, device=cuda).to(qd)
    kl, kw = i32(lens), dict(k_scale=ks, v_scale=vs)
    if form == "workspace":
        kw["workspace"] = b200decode.DecodeWorkspace(cuda, 64 << 20)
    call = lambda: b200decode.cross_attention(q[:, None] if form == "B1HD" else q, k, v, kl, bt, **kw)  # noqa: E731
    out, lse = call()
    if form == "captured":
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = call()
        g.replay()
    torch.cuda.synchronize()
    b200decode.check_device_status(kw.get("workspace"))
    for b, n in enumerate(lens):
        r = attend(q[b:b + 1].double(), gather(k, ks, bt[b], n, "NHD"), gather(v, vs, bt[b], n, "NHD"), d ** -0.5, kv)
        check(out.reshape(4, hq, d)[b:b + 1], r[0], r[2], u_of(qd), "out")
        check_lse(lse.reshape(4, hq)[b:b + 1], r[1], r[3])


@pytest.mark.parametrize("P", [16, 5])
@pytest.mark.parametrize("starts", [[0, 12, 5, 20], [3, 1, 1, 20], [0, 20, 20, 19]])
def test_descending_starts_are_reported(cuda, P, starts):
    """Starts that descend would give tokens to two groups: nothing is written,
    and the status says so."""
    gen, k, v, _, _, bt = paged(cuda, 310, [96, 64, 40], P, 2, 64, BF)
    q = torch.randn(20, 4, 64, generator=gen, device=cuda).to(BF)
    kl, st = i32([96, 64, 40]), i32(starts)
    ws = b200decode.DecodeWorkspace(cuda, 64 << 20)
    own, obt = i32([3] * 20), bt[:1].repeat(20, 1)
    for call in (lambda **kw: b200decode.cross_attention(q, k, v, kl, bt, workspace=ws, **kw),
                 lambda **kw: b200decode.decode_shared_prefix(q, k, v, kl, bt, own, obt, workspace=ws,
                                                              group_starts=kw.pop("query_starts"), **kw)):
        out, lse = torch.full_like(q, 7.0), torch.full((20, 4), 7.0, device=cuda)
        call(query_starts=st, out=out, lse=lse)
        torch.cuda.synchronize()
        with pytest.raises(b200decode.B2DError) as e:
            b200decode.check_device_status(ws)
        assert e.value.code == -7
        assert (out == 7).all() and (lse == 7).all()
        a = call(query_starts=i32([0, 12, 15, 20]))
        b200decode.check_device_status(ws)
        b = call(query_starts=i32([0, 12, 15, 20]))
        assert torch.equal(a[0], b[0]) and torch.isfinite(a[0]).all()


def test_status_of_a_call_outlives_growth_by_the_next(cuda):
    gen, k, v, _, _, bt = paged(cuda, 315, [100, 50], 16, 2, 64, BF)
    q = torch.randn(70, 4, 64, generator=gen, device=cuda).to(BF)
    st, kl, bad = i32([0, 40, 70]), i32([100, 50]), bt.clone()
    bad[0, 2] = -1
    ws = b200decode.DecodeWorkspace(cuda)
    b200decode.cross_attention(q, k, v, kl, bad, query_starts=st, workspace=ws, num_ctas=2)
    size = ws.nbytes
    b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws, num_ctas=300)
    assert ws.nbytes > size
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -7
    b200decode.check_device_status(ws)


def test_buffer_of_a_captured_decode_outlives_growth(cuda):
    """A graph that holds a workspace's buffer replays into memory that is its
    own, also after a later call made the workspace grow."""
    gen, k, v, _, _, bt = paged(cuda, 360, [5000, 3000], 16, 2, 128, BF)
    q, kl = torch.randn(2, 8, 128, generator=gen, device=cuda).to(BF), i32([5000, 3000])
    ws = b200decode.DecodeWorkspace(cuda)
    want = b200decode.decode(q, k, v, kl, bt, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = b200decode.decode(q, k, v, kl, bt, workspace=ws)
    old = ws.buf.data_ptr()
    many = torch.randn(300, 8, 128, generator=gen, device=cuda).to(BF)
    b200decode.cross_attention(many, k, v, kl, bt, query_starts=i32([0, 100, 300]), workspace=ws, num_ctas=600)
    assert ws.buf.data_ptr() != old
    fill = [torch.full((1 << 20,), 77, dtype=torch.uint8, device=cuda) for _ in range(8)]
    assert all(f.data_ptr() != old for f in fill)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert all((f == 77).all() for f in fill)
    b200decode.check_device_status(ws)


# ---------------------------------------------------------------- rows without mass

def minus_infinity(k, P, layout, row, n):
    """Makes every score of a row's first n tokens -inf for positive queries."""
    for pos in range(n):
        pg, off = int(row[pos // P]), pos % P
        if layout == "vllm":
            k[pg, :, 0, off, 0] = float("-inf")
        elif layout == "HND":
            k[pg, :, off, 0] = float("-inf")
        else:
            k[pg, off, :, 0] = float("-inf")


@pytest.mark.parametrize("num_ctas", [None, 1, 40])
@pytest.mark.parametrize("qd,hq,hkv,d,P,layout", [
    (BF, 8, 2, 128, 16, "NHD"), (HF, 4, 4, 64, 16, "HND"), (BF, 32, 2, 128, 16, "NHD"), (BF, 8, 2, 128, 5, "NHD"),
    (BF, 8, 2, 256, 16, "NHD"), (BF, 4, 2, 128, 16, "vllm")])
def test_shared_prefix_of_own_tokens_without_mass(cuda, qd, hq, hkv, d, P, layout, num_ctas):
    """Own tokens whose scores are all -inf (the first of them, all, all of a
    long sequence) weigh nothing beside the prefix; with no prefix: 0 and -inf."""
    plens, lens, starts = [150, 0], [40, 700, 3, 33, 40], [0, 3, 5]
    gen, k, v, ks, vs, both = paged(cuda, 320, plens + lens, P, hkv, d, qd, layout)
    pbt, bt = both[:2], both[2:]
    gone = [40, 700, 1, 20, 40]
    for b, n in enumerate(gone):
        minus_infinity(k, P, layout, bt[b], n)
    q = torch.rand(5, hq, d, generator=gen, device=cuda).add_(0.1).to(qd)
    kw = dict(kv_layout=layout, num_ctas=num_ctas)
    out, lse = b200decode.decode_shared_prefix(q, k, v, i32(plens), pbt, i32(lens), bt, group_starts=i32(starts), **kw)
    alone, alone_lse = b200decode.decode(q, k, v, i32(lens), bt, **kw)
    one, one_lse = b200decode.cross_attention(q, k, v, i32(lens), bt, **kw)
    torch.cuda.synchronize()
    b200decode.check_device_status()
    for b, n in enumerate(lens):
        kk, vv = gather(k, ks, bt[b], n, lay(layout, "k"))[gone[b]:], gather(v, vs, bt[b], n, lay(layout, "v"))[gone[b]:]
        own = attend(q[b:b + 1].double(), kk, vv, d ** -0.5, qd)
        r = own
        if b < 3:
            pre = attend(q[b:b + 1].double(), gather(k, ks, pbt[0], 150, lay(layout, "k")),
                         gather(v, vs, pbt[0], 150, lay(layout, "v")), d ** -0.5, qd)
            r = merge2(own, pre)
        check(out[b:b + 1], r[0], r[2], u_of(qd), "out")
        check_lse(lse[b:b + 1], r[1], r[3])
        for o, l in ((alone, alone_lse), (one, one_lse)):
            check(o[b:b + 1], own[0], own[2], u_of(qd), "own tokens alone")
            check_lse(l[b:b + 1], own[1], own[3])


@pytest.mark.parametrize("num_ctas", [None, 1, 7])
@pytest.mark.parametrize("P", [16, 5])
def test_shared_prefix_without_mass_keeps_a_nan_of_the_own_tokens(cuda, P, num_ctas):
    """A NaN among a sequence's own keys makes its rows NaN, also beside a
    prefix whose scores are all -inf; its neighbours are right."""
    gen, k, v, _, _, both = paged(cuda, 330, [200, 30, 30, 30], P, 2, 64, BF)
    pbt, bt = both[:1], both[1:]
    minus_infinity(k, P, "NHD", pbt[0], 200)
    k[bt[1, 17 // P].long(), 17 % P, :, 3] = float("nan")
    q = torch.rand(3, 4, 64, generator=gen, device=cuda).add_(0.1).to(BF)
    out, lse = b200decode.decode_shared_prefix(q, k, v, i32([200]), pbt, i32([30] * 3), bt, num_ctas=num_ctas)
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    for b in (0, 2):
        r = attend(q[b:b + 1].double(), gather(k, None, bt[b], 30, "NHD"), gather(v, None, bt[b], 30, "NHD"), 0.125, BF)
        check(out[b:b + 1], r[0], r[2] * (1 + 2.0 ** -11), u_of(BF), "out")
        check_lse(lse[b:b + 1], r[1], r[3] + 2.0 ** -20 * (1 + r[1].abs()))


# ---------------------------------------------------------------- small weights

@pytest.mark.parametrize("num_ctas", [None, 1])
@pytest.mark.parametrize("score", [16.875, 18.0])
@pytest.mark.parametrize("kv,d,P", [(HF, 64, 16), (F8, 128, 16), (HF, 128, 5), (HF, 256, 16), (F8, 64, 5)])
def test_many_weights_far_below_the_largest(cuda, kv, d, P, score, num_ctas):
    """One key holds nearly all the weight and a value of 0, as an attention
    sink does; thousands of equal weights of e^-score beside it make the whole
    output.  In fp16 as they are, they would be multiples of 2^-24 of a value
    near one of them (or 0); the kernels scale them by 2^7 or more first, so each
    is off by at most 2^-32 of the largest."""
    n = 20000
    gen, k, v, _, _, bt = paged(cuda, 340, [n, n, 16], P, 1, d, kv)
    scale = 1.0 if score == 18.0 else 0.9375                  # (both exact, in e4m3 too)
    k.copy_(torch.zeros(k.shape, device=cuda).to(kv))
    v.copy_(torch.ones(v.shape, device=cuda).to(kv))
    sink, zero = torch.zeros(1, d, device=cuda), torch.zeros(1, d, device=cuda)
    sink[0, 0] = 18.0
    for b, pos in ((0, 0), (1, n - 3), (2, 1)):
        pg, off = bt[b, pos // P].long(), pos % P
        k[pg, off] = sink.to(kv)
        v[pg, off] = zero.to(kv)
    q = torch.zeros(9, 2, d, device=cuda, dtype=HF)
    q[:, :, 0] = 1

    def near(out, lse, r):
        u = 2.0 ** -11
        # scores are exact; sums of n terms, powers and the join in fp32: n 2^-24 + 2^-17
        tol = r[0].abs() * (u + n * 2.0 ** -24 + 2.0 ** -17) + n * 2.0 ** -32
        check(out, r[0], tol, u_of(HF), "out")
        check_lse(lse, r[1], r[3])

    ref = [attend(q[:1].double(), gather(k, None, bt[b], m, "NHD"), gather(v, None, bt[b], m, "NHD"), scale, kv)
           for b, m in ((0, n), (1, n), (2, 16))]
    out, lse = b200decode.cross_attention(q, k, v, i32([n, n, 16]), bt, scale, query_starts=i32([0, 4, 6, 9]),
                                          num_ctas=num_ctas)
    for b, (lo, hi) in enumerate(((0, 4), (4, 6), (6, 9))):
        for t in range(lo, hi):
            near(out[t:t + 1], lse[t:t + 1], ref[b])
    # the long tail in the prefix, and in the own tokens
    both = merge2(ref[0], ref[2])
    for pl, ol, pb, ob in ((n, 16, bt[:1], bt[2:]), (16, n, bt[2:], bt[:1])):
        out, lse = b200decode.decode_shared_prefix(q, k, v, i32([pl]), pb, i32([ol] * 9), ob.repeat(9, 1), scale,
                                                   num_ctas=num_ctas)
        for t in range(9):
            near(out[t:t + 1], lse[t:t + 1], both)


# ---------------------------------------------------------------- errors that a bound for each element does not see

def spread(got, q, k, v, scale, kv, qd):
    """Mean of (error / s)^2 over all elements, s^2 = (u_out out)^2 + u_p^2 sum_j (p_j v_j)^2.
    The rounding of out is off by at most u_out |out|, and each weight, rounded
    to 16 bits by itself, by at most u_p of its size, with no common sign: were
    all at their limits the mean would be 1, as they are spread it is about 1/3.
    (fp32 errors of scores and sums are under 2^-18 of a weight.)  A part that is
    lost, misplaced or misweighted shows long before it passes the bound for
    each element, which adds up all weights' errors."""
    T, hq, d = q.shape
    grp = hq // k.shape[1]
    k, v = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
    p = torch.softmax(torch.einsum("thd,lhd->thl", q.double(), k) * scale, -1)
    out = torch.einsum("thl,lhd->thd", p, v)
    u_p = 2.0 ** -8 if kv == BF else 2.0 ** -11
    s2 = (u_of(qd) * out) ** 2 + u_p ** 2 * torch.einsum("thl,lhd->thd", p ** 2, v ** 2)
    return float((((got.double() - out) ** 2) / s2).mean())


@pytest.mark.parametrize("num_ctas", [None, 5])
@pytest.mark.parametrize("qd,kv,hq,hkv,d,P", [(BF, BF, 8, 2, 128, 16), (HF, HF, 4, 4, 64, 64), (BF, F8, 16, 2, 128, 16),
                                              (BF, BF, 8, 2, 128, 5), (HF, HF, 4, 1, 256, 16)])
def test_spread_of_errors(cuda, qd, kv, hq, hkv, d, P, num_ctas):
    lens, tq = [9000, 1000, 130], [40, 140, 9]
    gen, k, v, ks, vs, bt = paged(cuda, 370, lens, P, hkv, d, kv)
    q = torch.randn(189, hq, d, generator=gen, device=cuda).to(qd)
    out, _ = b200decode.cross_attention(q, k, v, i32(lens), bt, query_starts=i32([0, 40, 180, 189]), k_scale=ks,
                                        v_scale=vs, num_ctas=num_ctas)
    for b, (lo, hi) in enumerate(((0, 40), (40, 180), (180, 189))):
        kk, vv = gather(k, ks, bt[b], lens[b], "NHD"), gather(v, vs, bt[b], lens[b], "NHD")
        assert spread(out[lo:hi], q[lo:hi], kk, vv, d ** -0.5, kv, qd) < 1
    # own tokens behind a prefix: request 0's keys, then request 1's or 2's
    own = [1 + i % 2 for i in range(20)]
    out, _ = b200decode.decode_shared_prefix(q[:20], k, v, i32(lens[:1]), bt[:1], i32([lens[b] for b in own]),
                                             bt[torch.tensor(own)], k_scale=ks, v_scale=vs, num_ctas=num_ctas)
    for b in (1, 2):
        kk, vv = (torch.cat([gather(c, s, bt[x], lens[x], "NHD") for x in (0, b)]) for c, s in ((k, ks), (v, vs)))
        assert spread(out[b - 1:20:2], q[b - 1:20:2], kk, vv, d ** -0.5, kv, qd) < 1


@pytest.mark.parametrize("num_ctas", [None, 3, 29])
@pytest.mark.parametrize("kv,d,P", [(BF, 128, 16), (HF, 64, 48), (F8, 128, 16), (BF, 128, 5), (BF, 192, 16)])
def test_every_border_token_counts_once(cuda, kv, d, P, num_ctas):
    """V is 1 in a dim of its own for a few tokens, at the borders of pages,
    chunks and sequences, and 0 elsewhere: that dim of out is the token's own
    weight, off by its two roundings and no more."""
    n = 3000
    lens = [n, 130]
    gen, k, v, ks, _, bt = paged(cuda, 380, lens, P, 2, d, kv)
    at = sorted({x for c in (0, P, 128, 256, 1024, 1536, 2048, n - 1, n - P) for x in (c - 1, c, c + 1) if 0 <= x < n})
    at += [x for x in range(700, n, 131) if x not in at][:d - len(at)]
    v.copy_(torch.zeros(v.shape, device=cuda).to(kv))
    for i, pos in enumerate(at):
        row = torch.zeros(2, d, device=cuda)
        row[:, i] = 1
        v[bt[0, pos // P].long(), pos % P] = row.to(kv)
        if pos < 130:
            v[bt[1, pos // P].long(), pos % P] = row.to(kv)
    q = (0.3 * torch.randn(70, 8, d, generator=gen, device=cuda)).to(HF if kv == HF else BF)

    def weights(qq, keys, parts, got):
        s = torch.einsum("thd,lhd->thl", qq.double(), keys.repeat_interleave(4, 1)) * d ** -0.5
        p, want = torch.softmax(s, -1), torch.zeros(qq.shape, dtype=torch.float64, device=cuda)
        for base, length in parts:
            for i, pos in enumerate(at):
                if pos < length:
                    want[..., i] += p[..., base + pos]
        # a weight rounded to 16 bits (fp16: scaled, so 2^-32 of the largest at least); its score and the
        # maximum off by ds each (serving_ref.py); powers, sums and the join in fp32; out rounded by check()
        u_p, least = (2.0 ** -8, 0.0) if kv == BF else (2.0 ** -11, 2.0 ** -32)
        s_abs = torch.einsum("thd,lhd->thl", qq.double().abs(), keys.abs().repeat_interleave(4, 1)).amax(-1) * d ** -0.5
        ds = 2.0 ** -24 * (d + 4) * s_abs[..., None]
        check(got, want, want * (u_p + 2 * ds + keys.shape[0] * 2.0 ** -24 + 2.0 ** -17) + least, u_of(got.dtype), "weights")

    ks = ks if kv == F8 else None
    k0, k1 = (gather(k, ks, bt[b], m, "NHD") for b, m in ((0, n), (1, 130)))
    out, _ = b200decode.cross_attention(q, k, v, i32(lens), bt, query_starts=i32([0, 60, 70]), k_scale=ks,
                                        num_ctas=num_ctas)
    weights(q[:60], k0, [(0, n)], out[:60])
    weights(q[60:], k1, [(0, 130)], out[60:])
    for pre, own in ((0, 1), (1, 0)):
        out, _ = b200decode.decode_shared_prefix(q[:33], k, v, i32([lens[pre]]), bt[pre:pre + 1], i32([lens[own]] * 33),
                                                 bt[own:own + 1].repeat(33, 1), k_scale=ks, num_ctas=num_ctas)
        both = torch.cat([(k0, k1)[pre], (k0, k1)[own]])
        weights(q[:33], both, [(0, lens[pre]), (lens[pre], lens[own])], out)


def test_first_capture_of_a_stream_leaves_eager_calls_a_zeroed_workspace(cuda):
    """A decode() captured on a stream that has no workspace yet; then, before
    any replay, steps on that stream whose blocks count themselves in the header."""
    gen, k, v, _, _, bt = paged(cuda, 390, [500, 300], 16, 2, 128, BF)
    q, kl = torch.randn(2, 8, 128, generator=gen, device=cuda).to(BF), i32([500, 300])
    want = b200decode.decode(q, k, v, kl, bt)
    b200decode.cross_attention(q, k, v, kl, bt, query_starts=i32([0, 1, 2]))
    B, P = 4000, 16
    lens, table = torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(B, 2, dtype=torch.int32, device=cuda)
    free, count = torch.arange(B, dtype=torch.int32, device=cuda), i32([B])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = b200decode.decode(q, k, v, kl, bt)
    with torch.cuda.stream(s):
        for _ in range(3):
            b200decode.plan_append(lens, table, free, count, P, seqlens_out=lens, free_count_out=count)
        s.synchronize()
        b200decode.check_device_status()
        assert (lens == 3).all() and int(count) == 0
        g.replay()
        s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("hkv,grp,d", [(8, 1, 256), (16, 4, 256), (7, 2, 256), (8, 4, 192)])
def test_wide_rows_of_many_heads(cuda, hkv, grp, d):
    """Eight KV heads of 256 dims do not fit a tile: narrower ones are taken
    (with a table wide enough that the batch alone would ask for wide tiles)."""
    lens, plen = [700, 1, 0, 333] * 16, 60
    gen, k, v, _, _, both = paged(cuda, 295, lens + [plen], 16, hkv, d, BF)
    bt, pbt = both[:64], both[64:, :4]
    q = torch.randn(64, hkv * grp, d, generator=gen, device=cuda).to(BF)
    wide = torch.zeros(64, 600, dtype=torch.int32, device=cuda)
    wide[:, :bt.shape[1]] = bt
    got = [b200decode.decode(q, k, v, i32(lens), wide), b200decode.cross_attention(q, k, v, i32(lens), wide),
           b200decode.decode_shared_prefix(q, k, v, i32([plen]), pbt, i32(lens), wide)]
    torch.cuda.synchronize()
    b200decode.check_device_status()
    for b in (0, 1, 2, 3, 40, 63):
        part = [attend(q[b:b + 1].double(), gather(k, None, r, m, "NHD"), gather(v, None, r, m, "NHD"), d ** -0.5, BF)
                for r, m in ((bt[b], lens[b]), (pbt[0], plen))]
        for (out, lse), ref in zip(got, (part[0], part[0], merge2(*part))):
            check(out[b:b + 1], ref[0], ref[2], u_of(BF), "out")
            check_lse(lse[b:b + 1], ref[1], ref[3])


def test_shared_prefix_refuses_no_token(cuda):
    """q [B, 0, Hq, D] and [B, 2, Hq, D]: a ValueError of the call's own."""
    k = torch.zeros(4, 16, 2, 64, dtype=BF, device=cuda)
    kl, bt = i32([16, 16]), i32([[0], [1]])
    for n in (0, 2):
        q = torch.zeros(2, n, 4, 64, dtype=BF, device=cuda)
        with pytest.raises(ValueError, match="one query token"):
            b200decode.decode_shared_prefix(q, k, k, kl[:1], bt[:1], kl, bt)


# ---------------------------------------------------------------- every kernel

def draw(rng, i, pages, dims):
    """A random size, of the warp-level kernel where the pages or dims ask for it."""
    kv = rng.choice([BF, HF, F8])
    qd = HF if kv == HF else rng.choice([BF, HF]) if kv == F8 else BF
    d, P, layout = rng.choice(dims), rng.choice(pages), rng.choice(["NHD", "HND", "vllm"])
    if layout == "vllm" and (kv == F8 or P % 16):
        layout = "NHD"
    return kv, qd, rng.choice([1, 2, 3, 5, 8]), d, P, layout


@pytest.mark.parametrize("part", range(4))
def test_cross_fuzz_of_the_warp_level_kernel(cuda, part):
    import random
    rng = random.Random(100 + part)
    for i in range(15):
        kv, qd, hkv, d, P, layout = draw(rng, i, [1, 2, 5, 7, 8, 16, 24, 100, 128], [64, 128, 192, 256])
        grp = rng.choice([1, 2, 3, 5, 7, 8, 13, 16, 29, 32])
        lens = [rng.choice([0, 1, 31, 32, 33, 63, 64, 65, rng.randint(1, 700)]) for _ in range(rng.randint(1, 5))]
        tq = [rng.choice([0, 1, 2, rng.randint(1, 90)]) for _ in lens]
        starts = [sum(tq[:b]) for b in range(len(tq) + 1)]
        if starts[-1] == 0:
            continue
        gen, k, v, ks, vs, bt = paged(cuda, 400 + 20 * part + i, lens, P, hkv, d, kv, layout)
        q = torch.randn(starts[-1], hkv * grp, d, generator=gen, device=cuda).to(qd)
        out, lse = b200decode.cross_attention(q, k, v, i32(lens), bt, query_starts=i32(starts), k_scale=ks, v_scale=vs,
                                              kv_layout=layout, num_ctas=rng.choice([None, None, 1, 2, 13, 300]))
        for b, n in enumerate(lens):
            s = slice(starts[b], starts[b + 1])
            if tq[b]:
                r = attend(q[s].double(), gather(k, ks, bt[b], n, lay(layout, "k")),
                           gather(v, vs, bt[b], n, lay(layout, "v")), d ** -0.5, kv)
                check(out[s], r[0], r[2], u_of(qd), f"{i}: out")
                check_lse(lse[s], r[1], r[3])
    b200decode.check_device_status()


@pytest.mark.parametrize("part", range(6))
def test_shared_fuzz(cuda, part):
    import random
    rng = random.Random(200 + part)
    for i in range(15):
        kv, qd, hkv, d, P, layout = draw(rng, i, [16, 16, 32, 48, 64, 112, 256, 1, 5, 8, 24], [64, 128, 128, 256])
        grp = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
        B, G = rng.randint(1, 40), rng.choice([1, 1, 2, 5])
        cuts = sorted(rng.randint(0, B) for _ in range(G + 1))
        plens = [rng.choice([0, 1, 127, 128, 129, rng.randint(1, 900)]) for _ in range(G)]
        lens = [rng.choice([0, 1, 15, 16, 17, rng.randint(1, 300)]) for _ in range(B)]
        gen, k, v, ks, vs, both = paged(cuda, 600 + 20 * part + i, plens + lens, P, hkv, d, kv, layout)
        pbt, bt = both[:G], both[G:]
        q = torch.randn(B, hkv * grp, d, generator=gen, device=cuda).to(qd)
        out, lse = b200decode.decode_shared_prefix(q, k, v, i32(plens), pbt, i32(lens), bt, group_starts=i32(cuts),
                                                   k_scale=ks, v_scale=vs, kv_layout=layout,
                                                   num_ctas=rng.choice([None, None, 1, 3, 50, 400]))
        for b in range(B):
            one = lambda row, n: attend(q[b:b + 1].double(), gather(k, ks, row, n, lay(layout, "k")),   # noqa: E731
                                        gather(v, vs, row, n, lay(layout, "v")), d ** -0.5, kv)
            r = one(bt[b], lens[b])
            for g in range(G):
                if cuts[g] <= b < cuts[g + 1]:
                    r = merge2(r, one(pbt[g], plens[g]))
            check(out[b:b + 1], r[0], r[2], u_of(qd), f"{i}: out {b}")
            check_lse(lse[b:b + 1], r[1], r[3])
    b200decode.check_device_status()


@pytest.mark.parametrize("d,P,layout,kv", [(128, 5, "NHD", BF), (256, 16, "HND", HF), (64, 7, "NHD", F8), (128, 16, "vllm", BF)])
@pytest.mark.parametrize("num_ctas", [None, 1, 9])
def test_warp_level_kernel_with_odd_values(cuda, d, P, layout, kv, num_ctas):
    """NaN and infinity in a valid key stay with their request and KV head;
    a page out of range is read as page 0 and reported; scales of either sign."""
    lens, tq = [300, 150, 200], [40, 9, 30]
    gen, k, v, ks, vs, bt = paged(cuda, 395, lens, P, 2, d, kv, layout)
    if kv == F8:
        ks[1] = -ks[1]
    qd = HF if kv == HF else BF
    q = torch.rand(79, 8, d, generator=gen, device=cuda).add_(0.1).to(qd)
    st, kl = i32([0, 40, 49, 79]), i32(lens)
    ws = b200decode.DecodeWorkspace(cuda, 64 << 20)
    call = lambda kk, tt, scale: b200decode.cross_attention(   # noqa: E731
        q, kk, v, kl, tt, scale, query_starts=st, k_scale=ks, v_scale=vs, kv_layout=layout, num_ctas=num_ctas, workspace=ws)
    for scale in (-0.05, 0.0, d ** -0.5):
        out, lse = call(k, bt, scale)
        for b, (lo, hi) in enumerate(((0, 40), (40, 49), (49, 79))):
            r = attend(q[lo:hi].double(), gather(k, ks, bt[b], lens[b], lay(layout, "k")),
                       gather(v, vs, bt[b], lens[b], lay(layout, "v")), scale, kv)
            check(out[lo:hi], r[0], r[2], u_of(qd), "out")
            check_lse(lse[lo:hi], r[1], r[3])
    b200decode.check_device_status(ws)
    for pos in (0, 77, 299):
        for value in (float("nan"), float("inf")):
            if kv == F8 and value == float("inf"):
                continue
            bad = k.clone()
            raw = bad.view(torch.uint8) if kv == F8 else bad
            pg, off = int(bt[0, pos // P]), pos % P
            at = (pg, 1, 0, off, 5) if layout == "vllm" else (pg, 1, off, 5) if layout == "HND" else (pg, off, 1, 5)
            raw[at] = 0x7F if kv == F8 else value
            got, _ = call(bad, bt, d ** -0.5)
            assert torch.isnan(got[:40, 4:]).all() and torch.equal(got[:40, :4], out[:40, :4])
            assert torch.equal(got[40:], out[40:])
    for page in (-1, k.shape[0], 2 ** 31 - 1):
        wrong, zero = bt.clone(), bt.clone()
        wrong[1, 2], zero[1, 2] = page, 0
        got, _ = call(k, wrong, d ** -0.5)
        with pytest.raises(b200decode.B2DError) as e:
            b200decode.check_device_status(ws)
        assert e.value.code == -7
        assert torch.equal(got, call(k, zero, d ** -0.5)[0])
