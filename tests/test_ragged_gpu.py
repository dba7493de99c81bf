"""decode_shared_prefix, cross_attention and merge_states on the GPU, against a
64-bit reference with derived bounds (serving_ref.py)."""
import pytest
import torch

import b200decode
from b200decode import _lib
from serving_ref import attend, caches, check, check_lse, gather, merge2, tables, u_of

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(device, seed, lens, P, hkv, d, kv, layout, extra_pages=3):
    """Paged keys of sequences `lens`, pages in random order, a few unused;
    slots past a sequence's end hold NaN."""
    gen = torch.Generator(device=device).manual_seed(seed)
    pages = sum((n + P - 1) // P for n in lens) + extra_pages
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    k, v, ks, vs = caches(gen, device, pages, P, hkv, d, kv, layout)
    bt, _ = tables(lens, P, perm, 0)
    for i, n in enumerate(lens):
        if n % P:
            pg, off = int(bt[i, n // P]), n % P
            for c, is_v in ((k, False), (v, True)):
                raw = c.view(torch.uint8) if c.dtype == F8 else c
                bad = 0x7F if c.dtype == F8 else float("nan")
                if layout == "NHD":
                    raw[pg, off:] = bad
                elif layout == "HND":
                    raw[pg, :, off:] = bad
                elif is_v:
                    raw[pg, :, :, off:] = bad
                else:
                    raw[pg, :, :, off:] = bad
    return gen, k, v, ks, vs, bt.to(device)


def lay(layout, which):
    return f"vllm_{which}" if layout == "vllm" else layout


def cross_reference(q, k, v, ks, vs, bt, starts, lens, scale, layout):
    parts = []
    for b, n in enumerate(lens):
        kk, vv = gather(k, ks, bt[b], n, lay(layout, "k")), gather(v, vs, bt[b], n, lay(layout, "v"))
        parts.append(attend(q[starts[b]:starts[b + 1]].double(), kk, vv, scale, k.dtype))
    return [torch.cat(x) for x in zip(*parts)]


CROSS = [
    # q dtype, kv dtype, Hq, Hkv, D, P, layout, query counts, key counts
    (BF, BF, 8, 8, 64, 16, "NHD", [3, 5], [300, 70]),
    (BF, BF, 32, 8, 128, 16, "NHD", [1, 40, 0, 129, 7], [1, 129, 50, 1000, 0]),
    (HF, HF, 16, 4, 128, 64, "HND", [70, 2, 33], [127, 128, 640]),
    (BF, F8, 32, 8, 128, 16, "NHD", [17, 64, 1], [255, 513, 31]),
    (HF, F8, 6, 2, 64, 32, "HND", [100, 11], [99, 1025]),
    (BF, BF, 14, 2, 128, 48, "NHD", [50, 19], [700, 95]),          # group 7, page 48
    (HF, HF, 5, 1, 64, 80, "NHD", [200, 1], [161, 1]),             # group 5, page 80
    (BF, BF, 32, 1, 128, 128, "NHD", [9, 300], [2000, 129]),       # MQA
    (BF, BF, 4, 4, 128, 5, "NHD", [30, 65], [77, 6]),              # page 5
    (BF, F8, 8, 4, 128, 1, "NHD", [10], [130]),                    # page 1
    (BF, BF, 8, 2, 192, 16, "NHD", [20, 3], [100, 33]),
    (HF, HF, 8, 2, 256, 16, "HND", [66, 3], [100, 257]),
    (BF, F8, 8, 2, 256, 16, "NHD", [20, 3], [100, 33]),
    (BF, BF, 16, 4, 128, 16, "vllm", [65, 3], [300, 17]),
    (HF, HF, 8, 8, 64, 32, "vllm", [5, 70], [64, 99]),
]


@pytest.mark.parametrize("num_ctas", [None, 1, 7, 100])
@pytest.mark.parametrize("case", range(len(CROSS)))
def test_cross_attention(cuda, case, num_ctas):
    qd, kv, hq, hkv, d, P, layout, tq, lens = CROSS[case]
    gen, k, v, ks, vs, bt = make(cuda, case, lens, P, hkv, d, kv, layout)
    starts = [0]
    for n in tq:
        starts.append(starts[-1] + n)
    T = starts[-1]
    q = torch.randn(T + 2, hq, d, generator=gen, device=cuda).to(qd)   # two rows behind the last request
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    kl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0)
    lse = torch.full((T + 2, hq), 7.0, device=cuda)
    b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, k_scale=ks, v_scale=vs, out=out, lse=lse,
                               kv_layout=layout, num_ctas=num_ctas)
    torch.cuda.synchronize()
    b200decode.check_device_status()
    ref = cross_reference(q, k, v, ks, vs, bt, starts, lens, d ** -0.5, layout)
    check(out[:T], ref[0], ref[2], u_of(qd), "out")
    check_lse(lse[:T], ref[1], ref[3])
    assert (out[T:] == 7).all() and (lse[T:] == 7).all()
    again, _ = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, k_scale=ks, v_scale=vs,
                                          kv_layout=layout, num_ctas=num_ctas)
    assert torch.equal(again[:T], out[:T])


@pytest.mark.parametrize("tq", [1, 2, 33])
def test_cross_dense_form(cuda, tq):
    """[B, Tq, Hq, D] (and [B, Hq, D]) without query_starts, strided q and out."""
    lens = [200, 1, 77]
    gen, k, v, _, _, bt = make(cuda, 40 + tq, lens, 16, 4, 128, BF, "NHD")
    big = torch.randn(3, tq, 20, 128, generator=gen, device=cuda).to(BF)
    q = big[:, :, 2:18]
    kl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    ref = cross_reference(q.reshape(-1, 16, 128), k, v, None, None, bt, [0, tq, 2 * tq, 3 * tq], lens, 0.3, "NHD")
    out, lse = b200decode.cross_attention(q, k, v, kl, bt, 0.3)
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    check(out.reshape(-1, 16, 128), ref[0], ref[2], u_of(BF), "out")
    check_lse(lse.reshape(-1, 16), ref[1], ref[3])
    if tq == 1:
        out, lse = b200decode.cross_attention(q[:, 0], k, v, kl, bt, 0.3)
        check(out, ref[0], ref[2], u_of(BF), "out")
        check_lse(lse, ref[1], ref[3])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
def test_cross_scales(cuda, scale):
    """Scales of either sign, none, and one that makes the softmax peaked."""
    lens, tq = [300, 140], [20, 37]
    gen, k, v, ks, vs, bt = make(cuda, 61, lens, 16, 2, 128, F8, "NHD")
    ks[1] = -ks[1]
    q = torch.randn(57, 8, 128, generator=gen, device=cuda).to(BF)
    st = torch.tensor([0, 20, 57], dtype=torch.int32, device=cuda)
    kl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out, lse = b200decode.cross_attention(q, k, v, kl, bt, scale, query_starts=st, k_scale=ks, v_scale=vs)
    ref = cross_reference(q, k, v, ks, vs, bt, [0, 20, 57], lens, scale, "NHD")
    check(out, ref[0], ref[2], u_of(BF), "out")
    check_lse(lse, ref[1], ref[3])


def test_cross_rising_scores(cuda):
    """Keys whose scores rise along the sequence by far more than a tile's
    spread, so that every tile moves the maximum; then falling."""
    n, d = 1500, 128
    gen, k, v, _, _, bt = make(cuda, 62, [n, n], 16, 1, d, BF, "NHD", extra_pages=0)
    q = torch.ones(200, 2, d, device=cuda, dtype=BF)
    ramp = torch.linspace(-3, 3, n, device=cuda)
    for b, r in ((0, ramp), (1, ramp.flip(0))):
        pos = torch.arange(n, device=cuda)
        k[bt[b, pos // 16].long(), pos % 16, 0] = (r[:, None] + 0.05 * torch.randn(n, d, generator=gen, device=cuda)).to(BF)
    st = torch.tensor([0, 100, 200], dtype=torch.int32, device=cuda)
    kl = torch.tensor([n, n], dtype=torch.int32, device=cuda)
    for ctas in (None, 1):
        out, lse = b200decode.cross_attention(q, k, v, kl, bt, 0.5, query_starts=st, num_ctas=ctas)
        ref = cross_reference(q, k, v, None, None, bt, [0, 100, 200], [n, n], 0.5, "NHD")
        check(out, ref[0], ref[2], u_of(BF), "out")
        check_lse(lse, ref[1], ref[3])


def test_cross_minus_infinity_scores(cuda):
    """Tiles whose scores are all -inf (keys of -inf) add nothing; a row of
    such keys alone gives 0 and -inf."""
    n, d = 400, 64
    gen, k, v, _, _, bt = make(cuda, 63, [n, 64], 16, 1, d, BF, "NHD", extra_pages=0)
    k[bt[0, :12].long(), :, 0, 0] = float("-inf")      # tokens 0 .. 191
    k[bt[1, :4].long(), :, 0, 0] = float("-inf")
    q = torch.rand(70, 1, d, generator=gen, device=cuda).add_(0.1).to(BF)
    st = torch.tensor([0, 66, 70], dtype=torch.int32, device=cuda)
    kl = torch.tensor([n, 64], dtype=torch.int32, device=cuda)
    for ctas in (None, 1):
        out, lse = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, num_ctas=ctas)
        kk, vv = gather(k, None, bt[0], n, "NHD")[192:], gather(v, None, bt[0], n, "NHD")[192:]
        ref = attend(q[:66].double(), kk, vv, d ** -0.5, BF)
        check(out[:66], ref[0], ref[2], u_of(BF), "out")
        check_lse(lse[:66], ref[1], ref[3])
        assert (out[66:] == 0).all() and torch.isneginf(lse[66:]).all()


@pytest.mark.parametrize("kv", [BF, HF, F8])
@pytest.mark.parametrize("num_ctas", [None, 1, 9])
def test_cross_nan_and_infinity_in_keys(cuda, kv, num_ctas):
    """A key of NaN (or one whose score is +inf) among a request's keys makes
    its rows NaN, on its KV head and nowhere else; in a masked place it changes
    nothing (make() has NaN there)."""
    lens, tq, d = [500, 300, 200], [40, 9, 70], 128
    gen, k, v, _, _, bt = make(cuda, 64, lens, 16, 2, d, kv, "NHD", extra_pages=0)
    q = torch.rand(119, 4, d, generator=gen, device=cuda).add_(0.1).to(BF if kv != HF else HF)
    st = torch.tensor([0, 40, 49, 119], dtype=torch.int32, device=cuda)
    kl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    clean, _ = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, num_ctas=num_ctas)
    assert torch.isfinite(clean).all()
    for pos in (0, 77, 333, 499):
        bad = k.clone()
        raw, code = (bad.view(torch.uint8), 0x7F) if kv == F8 else (bad, float("nan") if pos != 77 else float("inf"))
        raw[bt[0, pos // 16].long(), pos % 16, 1, 5] = code
        out, lse = b200decode.cross_attention(q, bad, v, kl, bt, query_starts=st, num_ctas=num_ctas)
        assert torch.isnan(out[:40, 2:]).all() and torch.isnan(lse[:40, 2:]).all(), pos
        assert torch.equal(out[:40, :2], clean[:40, :2]) and torch.equal(out[40:], clean[40:]), pos


@pytest.mark.parametrize("num_ctas", [1, 2, 3, 5, 11])
@pytest.mark.parametrize("d,P", [(64, 16), (128, 5)])
def test_cross_several_items_per_block(cuda, d, P, num_ctas):
    """Many tiles of long sequences to a block (the order of items on the work
    line changes with their number per block), odd tile counts, a cut or none."""
    lens, tq = [2100, 2048, 10, 4000], [700, 130, 3, 260]
    gen, k, v, _, _, bt = make(cuda, 80, lens, P, 3, d, BF, "NHD")
    starts = [0]
    for n in tq:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], 6, d, generator=gen, device=cuda).to(BF)
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    kl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out, lse = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, num_ctas=num_ctas)
    ref = cross_reference(q, k, v, None, None, bt, starts, lens, d ** -0.5, "NHD")
    check(out, ref[0], ref[2], u_of(BF), "out")
    check_lse(lse, ref[1], ref[3])


def test_cross_fuzz(cuda):
    """Random shapes of every kind against the reference."""
    import random
    rng = random.Random(11)
    for i in range(60):
        kv = rng.choice([BF, HF, F8])
        qd = HF if kv == HF else rng.choice([BF, HF]) if kv == F8 else BF
        hkv, grp, d = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3, 5, 6, 7, 8, 16, 31, 32]), rng.choice([64, 128])
        P, layout = rng.choice([16, 32, 48, 64, 112, 128, 256]), rng.choice(["NHD", "HND"])
        B = rng.randint(1, 6)
        lens = [rng.choice([0, 1, 63, 64, 65, 127, 128, 129, rng.randint(1, 900)]) for _ in range(B)]
        tq = [rng.choice([0, 1, 2, rng.randint(1, 150)]) for _ in range(B)]
        gen, k, v, ks, vs, bt = make(cuda, 1000 + i, lens, P, hkv, d, kv, layout)
        starts = [0]
        for n in tq:
            starts.append(starts[-1] + n)
        if starts[-1] == 0:
            continue
        q = torch.randn(starts[-1], hkv * grp, d, generator=gen, device=cuda).to(qd)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        out, lse = b200decode.cross_attention(q, k, v, i32(lens), bt, query_starts=i32(starts), k_scale=ks, v_scale=vs,
                                              kv_layout=layout, num_ctas=rng.choice([None, None, 2, 13, 300]))
        ref = cross_reference(q, k, v, ks, vs, bt, starts, lens, d ** -0.5, layout)
        check(out, ref[0], ref[2], u_of(qd), f"{i} out")
        check_lse(lse, ref[1], ref[3])
    b200decode.check_device_status()


def shared_reference(q, k, v, ks, vs, pbt, plens, bt, lens, starts, scale, layout):
    out = []
    for b in range(q.shape[0]):
        parts = [attend(q[b:b + 1].double(), gather(k, ks, bt[b], lens[b], lay(layout, "k")),
                        gather(v, vs, bt[b], lens[b], lay(layout, "v")), scale, k.dtype)]
        for g in range(len(plens)):
            if starts[g] <= b < starts[g + 1]:
                parts.append(attend(q[b:b + 1].double(), gather(k, ks, pbt[g], plens[g], lay(layout, "k")),
                                    gather(v, vs, pbt[g], plens[g], lay(layout, "v")), scale, k.dtype))
        out.append(parts[0] if len(parts) == 1 else merge2(*parts))
    return [torch.cat(x) for x in zip(*out)]


SHARED = [
    # q, kv, Hq, Hkv, D, P, layout, group starts, prefix lengths, own lengths
    (BF, BF, 32, 8, 128, 16, "NHD", [0, 4], [1024], [16, 256, 0, 1]),
    (BF, F8, 32, 8, 128, 16, "NHD", [0, 70], [999], [i % 40 for i in range(70)]),
    (HF, HF, 8, 8, 64, 32, "HND", [0, 1, 1, 9, 20], [5, 700, 128, 0], [3 * i for i in range(23)]),  # 3 ungrouped
    (BF, BF, 14, 2, 128, 48, "NHD", [0, 33], [577], [20] * 33),
    (BF, BF, 64, 2, 128, 64, "NHD", [0, 2, 12], [3000, 65], [100] * 12),
    (HF, F8, 12, 4, 64, 16, "NHD", [0, 40], [129], [9] * 40),
    (BF, BF, 8, 2, 256, 16, "NHD", [0, 5], [130], [33] * 5),
    (BF, BF, 8, 2, 192, 16, "NHD", [0, 5], [130], [33] * 5),
    (BF, BF, 8, 2, 128, 4, "NHD", [0, 20], [130], [33] * 20),
    (BF, BF, 8, 2, 128, 16, "vllm", [0, 20], [130], [33] * 20),
]


@pytest.mark.parametrize("num_ctas", [None, 1, 7, 100])
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_decode_shared_prefix(cuda, case, num_ctas):
    qd, kv, hq, hkv, d, P, layout, starts, plens, lens = SHARED[case]
    gen, k, v, ks, vs, both = make(cuda, 100 + case, plens + lens, P, hkv, d, kv, layout)
    pbt, bt = both[:len(plens)], both[len(plens):]
    q = torch.randn(len(lens), hq, d, generator=gen, device=cuda).to(qd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out, lse = b200decode.decode_shared_prefix(q, k, v, i32(plens), pbt, i32(lens), bt, group_starts=i32(starts),
                                               k_scale=ks, v_scale=vs, kv_layout=layout, num_ctas=num_ctas)
    torch.cuda.synchronize()
    b200decode.check_device_status()
    ref = shared_reference(q, k, v, ks, vs, pbt, plens, bt, lens, starts, d ** -0.5, layout)
    check(out, ref[0], ref[2], u_of(qd), "out")
    check_lse(lse, ref[1], ref[3])


@pytest.mark.parametrize("plens,starts", [([100], [0, 6]), ([100, 0], [1, 4, 6])])
def test_shared_prefix_shorter_than_own_tokens(cuda, plens, starts):
    """The prefix part is done long before the own tokens are: calls one after
    another in one workspace, eager and captured, equal calls on their own."""
    lens, d, P = [30000, 9000, 0, 12000, 17, 5000], 128, 16
    gen, k, v, _, _, both = make(cuda, 140, plens + lens, P, 2, d, BF, "NHD")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    pl, st, ol, pbt, bt = i32(plens), i32(starts), i32(lens), both[:len(plens)], both[len(plens):]
    qs = [torch.randn(6, 8, d, generator=gen, device=cuda).to(BF) for _ in range(4)]
    call = lambda q: b200decode.decode_shared_prefix(q, k, v, pl, pbt, ol, bt, group_starts=st)  # noqa: E731
    alone = []
    for q in qs:
        alone.append(call(q))
        torch.cuda.synchronize()
    ref = shared_reference(qs[0], k, v, None, None, pbt, plens, bt, lens, starts, d ** -0.5, "NHD")
    check(alone[0][0], ref[0], ref[2], u_of(BF), "out")
    check_lse(alone[0][1], ref[1], ref[3])
    # A wait limit below the default: one part after the other.
    limited = b200decode.decode_shared_prefix(qs[1], k, v, pl, pbt, ol, bt, group_starts=st, wait_limit_us=500000)
    assert all(torch.equal(x, y) for x, y in zip(limited, alone[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [call(q) for q in qs]
    for _ in range(5):
        eager = [call(q) for q in qs]
        graph.replay()
        torch.cuda.synchronize()
        for (o, l), (eo, el), (ho, hl) in zip(alone, eager, held):
            # (which warp merges a cut row's pieces does not change their order)
            assert torch.equal(o, eo) and torch.equal(l, el) and torch.equal(o, ho) and torch.equal(l, hl)


def test_shared_prefix_of_one_table(cuda):
    """One table whose rows begin with the same pages, cut by columns into the
    two tables; q [B, 1, Hq, D]; the result is decode()'s over whole rows."""
    P, B, n = 16, 6, 160
    lens = [n + x for x in (1, 30, 17, 64, 100, 5)]
    gen, k, v, _, _, bt = make(cuda, 120, lens, P, 2, 128, BF, "NHD")
    bt[:, :n // P] = bt[:1, :n // P]
    q = torch.randn(B, 1, 8, 128, generator=gen, device=cuda).to(BF)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    pl = torch.tensor([n], dtype=torch.int32, device=cuda)
    out, lse = b200decode.decode_shared_prefix(q, k, v, pl, bt[:1, :n // P], sl - n, bt[:, n // P:])
    ref = cross_reference(q[:, 0], k, v, None, None, bt, list(range(B + 1)), lens, 128 ** -0.5, "NHD")
    assert out.shape == q.shape
    # the join's weights: 2^-19 of sum softmax |v|, which is at most 2^8 of the bound
    check(out[:, 0], ref[0], ref[2] * (1 + 2.0 ** -11), u_of(BF), "out")
    check_lse(lse, ref[1], ref[3] + 2.0 ** -20 * (1 + ref[1].abs()))


def test_bad_pages_are_reported(cuda):
    """Page ids out of range are read as page 0 and reported."""
    gen, k, v, _, _, bt = make(cuda, 130, [100, 50], 16, 2, 64, BF, "NHD")
    q = torch.randn(70, 2, 64, generator=gen, device=cuda).to(BF)
    st = torch.tensor([0, 40, 70], dtype=torch.int32, device=cuda)
    kl = torch.tensor([100, 50], dtype=torch.int32, device=cuda)
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        b2 = bt.clone()
        b2[0, 3] = bad
        ws = b200decode.DecodeWorkspace(cuda)
        b200decode.cross_attention(q, k, v, kl, b2, query_starts=st, workspace=ws)
        with pytest.raises(b200decode.B2DError) as e:
            b200decode.check_device_status(ws)
        assert e.value.code == -7
        b3 = bt.clone()
        b3[0, 3] = 0
        out, _ = b200decode.cross_attention(q, k, v, kl, b2, query_starts=st, workspace=ws)
        ref, _ = b200decode.cross_attention(q, k, v, kl, b3, query_starts=st, workspace=ws)
        assert torch.equal(out, ref)


def test_lengths_and_starts_out_of_range_stay_inside(cuda):
    """Lengths are clamped to the table, starts to the tokens; negative ones to 0."""
    gen, k, v, _, _, bt = make(cuda, 131, [96, 64], 16, 2, 64, BF, "NHD")
    q = torch.randn(20, 2, 64, generator=gen, device=cuda).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out, _ = b200decode.cross_attention(q, k, v, i32([1000, -5]), bt, query_starts=i32([-3, 12, 99]))
    ref, _ = b200decode.cross_attention(q, k, v, i32([96, 0]), bt, query_starts=i32([0, 12, 20]))
    assert torch.equal(out, ref)


@pytest.mark.parametrize("shared", [False, True])
def test_captured_and_replayed(cuda, shared):
    """Calls captured without a workspace use the graph's own; inputs are
    refilled between replays; two graphs replayed at once on two streams."""
    lens, P, hkv, hq, d = [300, 170, 64], 16, 2, 8, 128
    gen, k, v, _, _, bt = make(cuda, 140, lens, P, hkv, d, BF, "NHD")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731

    def call(q, kl):
        if shared:
            return b200decode.decode_shared_prefix(q, k, v, kl[:1], bt[:1], kl[1:].repeat(20), bt[1:].repeat(20, 1))
        return b200decode.cross_attention(q, k, v, kl, bt, query_starts=i32([0, 25, 30, 40]))

    call(torch.zeros(40, hq, d, device=cuda, dtype=BF), i32(lens))
    graphs = []
    starts = i32([0, 25, 30, 40])
    for _ in range(2):
        q, kl = torch.zeros(40, hq, d, device=cuda, dtype=BF), i32(lens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if shared:
                res = call(q, kl)
            else:
                res = b200decode.cross_attention(q, k, v, kl, bt, query_starts=starts)
        graphs.append((g, q, kl, res))
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(4):
        want = []
        for i, (g, q, kl, res) in enumerate(graphs):
            q.copy_(torch.randn(40, hq, d, generator=gen, device=cuda))
            kl.copy_(i32([300 - step, 170 - 9 * i, 64 - 20 * step]))
            want.append([x.clone() for x in call(q, kl)])
        torch.cuda.synchronize()
        for s, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, _, res), w in zip(graphs, want):
            assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])


def test_two_streams_at_once(cuda):
    """The default workspace belongs to a stream: calls that overlap on two
    streams give what they give alone."""
    gen, k, v, _, _, bt = make(cuda, 150, [5000, 4000], 16, 2, 128, BF, "NHD")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    qs = [torch.randn(30 + i, 8, 128, generator=gen, device=cuda).to(BF) for i in range(2)]
    kl = i32([5000, 4000])
    st = [i32([0, 10, 30 + i]) for i in range(2)]
    alone = [b200decode.cross_attention(q, k, v, kl, bt, query_starts=s) for q, s in zip(qs, st)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(5):
        for s, q, t in zip(streams, qs, st):
            with torch.cuda.stream(s):
                got.append(b200decode.cross_attention(q, k, v, kl, bt, query_starts=t))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, alone[i % 2][0]) and torch.equal(l, alone[i % 2][1])


def test_workspace_held_by_a_graph_does_not_grow(cuda):
    gen, k, v, _, _, bt = make(cuda, 160, [300, 100], 16, 2, 64, BF, "NHD")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.randn(20, 2, 64, generator=gen, device=cuda).to(BF)
    kl, st = i32([300, 100]), i32([0, 12, 20])
    ws = b200decode.DecodeWorkspace(cuda, 200 << 20)
    want = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0])
    b200decode.check_device_status(ws)
    with pytest.raises(ValueError, match="cannot grow"):
        ws.ensure(ws.nbytes + 1)


def test_long_offsets(cuda):
    """Keys in pages whose element offset passes 32 bits."""
    P, hkv, d = 128, 8, 128
    pages = 2 ** 32 // (P * hkv * d) + 40            # 8.6 GB a cache
    k = torch.empty(pages, P, hkv, d, dtype=BF, device=cuda)
    v = torch.empty(pages, P, hkv, d, dtype=BF, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)
    ids = [pages - 1, 3, pages - 20, pages - 7]
    for i in ids:
        k[i] = torch.randn(P, hkv, d, generator=gen, device=cuda).to(BF)
        v[i] = torch.randn(P, hkv, d, generator=gen, device=cuda).to(BF)
    bt = torch.tensor([ids], dtype=torch.int32, device=cuda)
    q = torch.randn(50, 16, d, generator=gen, device=cuda).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out, lse = b200decode.cross_attention(q, k, v, i32([500]), bt, query_starts=i32([0, 50]))
    ref = cross_reference(q, k, v, None, None, bt, [0, 50], [500], d ** -0.5, "NHD")
    check(out, ref[0], ref[2], u_of(BF), "out")
    check_lse(lse, ref[1], ref[3])
    del k, v
    torch.cuda.empty_cache()


def test_many_groups(cuda):
    """More requests than one launch's chunk table holds."""
    B, P = 4200, 16
    lens = [(7 * i) % 40 for i in range(B)]
    gen, k, v, _, _, bt = make(cuda, 170, lens, P, 1, 64, BF, "NHD")
    tq = [(i * 5) % 3 for i in range(B)]
    starts = [0]
    for n in tq:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], 2, 64, generator=gen, device=cuda).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out, lse = b200decode.cross_attention(q, k, v, i32(lens), bt, query_starts=i32(starts))
    pick = list(range(0, B, 97)) + list(range(4090, 4110))
    for b in pick:
        if tq[b]:
            s = slice(starts[b], starts[b + 1])
            r = attend(q[s].double(), gather(k, None, bt[b], lens[b], "NHD"), gather(v, None, bt[b], lens[b], "NHD"),
                       0.125, BF)
            check(out[s], r[0], r[2], u_of(BF), "out")
            check_lse(lse[s], r[1], r[3])
    dense, _ = b200decode.cross_attention(q[:2 * B].reshape(B, 2, 2, 64) if q.shape[0] >= 2 * B else
                                          q.repeat(3, 1, 1)[:2 * B].reshape(B, 2, 2, 64), k, v, i32(lens), bt)
    qq = (q if q.shape[0] >= 2 * B else q.repeat(3, 1, 1))[:2 * B]
    for b in pick:
        r = attend(qq[2 * b:2 * b + 2].double(), gather(k, None, bt[b], lens[b], "NHD"),
                   gather(v, None, bt[b], lens[b], "NHD"), 0.125, BF)
        check(dense[b], r[0], r[2], u_of(BF), "out")


# ---------------------------------------------------------------- merge_states

@pytest.mark.parametrize("dtype,odt", [(BF, BF), (HF, HF), (torch.float32, torch.float32), (torch.float32, BF),
                                       (torch.float32, HF)])
@pytest.mark.parametrize("n,t,h,d", [(1, 1, 1, 8), (2, 5, 3, 64), (4, 33, 8, 128), (13, 2, 6, 576), (5, 7, 2, 1024)])
def test_merge_states(cuda, dtype, odt, n, t, h, d):
    gen = torch.Generator(device=cuda).manual_seed(n * 100 + d)
    o = torch.randn(n, t, h, d, generator=gen, device=cuda).to(dtype)
    l = 30 * torch.randn(n, t, h, generator=gen, device=cuda)
    gone = torch.rand(n, t, h, generator=gen, device=cuda) < 0.3
    l = l.masked_fill(gone, float("-inf"))
    o = o.masked_fill(gone[..., None], float("nan"))      # not read
    out = torch.empty(t, h, d, dtype=odt, device=cuda)
    out, lse = b200decode.merge_states(o, l, out=out)
    L = torch.logsumexp(l.double(), 0)
    w = torch.exp(l.double() - torch.where(torch.isinf(L), torch.zeros_like(L), L))
    oo = torch.where(gone[..., None], torch.zeros_like(o), o).double()
    ref = (w[..., None] * oo).sum(0)
    # weights: (lse_i - M) log2 e in fp32 is off by 2 roundings of at most its
    # size, of which only sizes under 30 ln-units carry weight: 60 * 2^-24 + 2^-21
    tol = (w[..., None] * oo.abs()).sum(0) * (2.0 ** -17 + n * 2.0 ** -22)
    check(out, ref, tol, u_of(odt), "out")
    check_lse(lse, L, 2.0 ** -21 * (1 + L.abs()) + 2.0 ** -20)


def test_merge_states_strided_in_place_of_decode(cuda):
    """Two decodes over halves of a cache, written into one buffer, merged:
    the decode over the whole."""
    gen, k, v, _, _, bt = make(cuda, 180, [320, 320], 16, 2, 128, BF, "NHD", extra_pages=0)
    q = torch.randn(2, 8, 128, generator=gen, device=cuda).to(BF)
    half = torch.tensor([160, 160], dtype=torch.int32, device=cuda)
    outs = torch.empty(2, 2, 8, 128, dtype=BF, device=cuda)
    lses = torch.empty(2, 2, 8, device=cuda)
    for i in range(2):
        b200decode.decode(q, k, v, half, bt[:, 10 * i:10 * i + 10].contiguous(), out=outs[i], lse=lses[i])
    wide = torch.zeros(2, 8, 256, dtype=BF, device=cuda)
    out, lse = b200decode.merge_states(outs, lses, out=wide[..., 64:192])
    ref = cross_reference(q, k, v, None, None, bt, [0, 1, 2], [320, 320], 128 ** -0.5, "NHD")
    # each half's out was rounded to bf16 on the way: 2^-8 sum softmax |v| more, at most ref[2] again
    check(out, ref[0], 2 * ref[2], u_of(BF), "out")
    check_lse(lse, ref[1], 2 * ref[3])
    assert (wide[..., :64] == 0).all() and (wide[..., 192:] == 0).all()


def test_wait_timeout_is_reported(cuda):
    """With the loads left out every bounded wait runs out; the call reports
    it, and the next call on the same workspace is right."""
    gen, k, v, _, _, bt = make(cuda, 190, [600, 300], 16, 2, 128, BF, "NHD")
    q = torch.randn(300, 8, 128, generator=gen, device=cuda).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    kl, st = i32([600, 300]), i32([0, 200, 300])
    ws = b200decode.DecodeWorkspace(cuda)
    want, _ = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws)
    b200decode.check_device_status(ws)
    b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws, flags=_lib.B2D_FLAG_TEST_NO_LOADS,
                               wait_limit_us=1000)
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -6
    got, _ = b200decode.cross_attention(q, k, v, kl, bt, query_starts=st, workspace=ws)
    b200decode.check_device_status(ws)
    assert torch.equal(got, want)
