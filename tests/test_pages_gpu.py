"""plan_append and release_pages on the GPU against a plain Python pool, and a
serving loop of all calls together."""
import pytest
import torch

import b200decode
from serving_ref import attend, check, check_lse, gather, merge2, u_of

pytestmark = pytest.mark.gpu


def pool_of(B, width, pages, P, lens, seed, device):
    """Requests of `lens` tokens on a shuffled pool."""
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    bt = torch.full((B, width), -9, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range((max(0, n) + P - 1) // P):
            bt[b, i] = perm.pop()
    free = torch.full((pages,), -5, dtype=torch.int32)
    free[:len(perm)] = torch.tensor(perm, dtype=torch.int32)
    return bt.to(device), free.to(device), torch.tensor([len(perm)], dtype=torch.int32, device=device)


def plain_append(lens, new, bt, free, count, P, max_tokens):
    bt, slots, starts, out = bt.tolist(), [], [0], []
    top = count
    for b, (L, n) in enumerate(zip(lens, new)):
        L, n = max(0, L), max(0, n)
        for pos in range(L, L + n):
            if pos % P == 0:
                top -= 1
                bt[b][pos // P] = int(free[top])
            slots.append(bt[b][pos // P] * P + pos % P)
        starts.append(len(slots))
        out.append(L + n)
    return slots + [-1] * (max_tokens - len(slots)), starts, out, top, bt


@pytest.mark.parametrize("B,P,hi,new_hi,spare", [
    (1, 16, 0, 1, 0), (1, 1, 40, 5, 3), (3, 16, 200, 1, 0), (64, 5, 100, 33, 10), (513, 16, 300, 4, 7),
    (1000, 32, 64, 40, 1), (5, 128, 5000, 9000, 2), (3000, 16, 40, 2, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_append(cuda, B, P, hi, new_hi, spare, in_place):
    g = torch.Generator().manual_seed(B * P)
    lens = torch.randint(0, hi + 1, (B,), generator=g).tolist()
    new = [1] * B if new_hi == 1 else torch.randint(0, new_hi + 1, (B,), generator=g).tolist()
    need = sum((L + n + P - 1) // P for L, n in zip(lens, new))
    width = (hi + new_hi) // P + 2
    bt, free, count = pool_of(B, width, need + 1, P, lens, B, cuda)
    if spare == 0 and need:
        # the pool has exactly the pages that the step takes
        exact = need - sum((L + P - 1) // P for L in lens)
        free[:exact] = free[int(count) - exact:int(count)].clone()
        count.fill_(exact)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = None if new_hi == 1 else torch.tensor(new, dtype=torch.int32, device=cuda)
    T = sum(new) + spare
    want = plain_append(lens, new, bt.cpu(), free.cpu(), int(count), P, T)
    before = free.clone()
    kw = dict(seqlens_out=sl, free_count_out=count) if in_place else {}
    plan = b200decode.plan_append(sl, bt, free, count, P, new_tokens=nt, max_tokens=T, **kw)
    torch.cuda.synchronize()
    b200decode.check_device_status()
    assert plan.slot_mapping.tolist() == want[0]
    assert plan.query_starts.tolist() == want[1]
    assert plan.cache_seqlens.tolist() == want[2]
    assert int(plan.free_count) == want[3]
    assert bt.tolist() == want[4]
    assert torch.equal(free, before)


@pytest.mark.parametrize("why", ["pages", "columns", "tokens", "count"])
@pytest.mark.parametrize("B", [4, 700])
def test_plan_append_that_does_not_fit_changes_nothing(cuda, why, B):
    P, lens = 16, [31] * B
    new = [3] * B
    width = 2 if why == "columns" else 3
    bt, free, count = pool_of(B, width, 5 * B, P, lens, 1, cuda)
    T = 3 * B - 1 if why == "tokens" else 3 * B + 2
    if why == "pages":
        count.fill_(B - 1)
    if why == "count":
        count.fill_(-4)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    nt = torch.tensor(new, dtype=torch.int32, device=cuda)
    ws = b200decode.DecodeWorkspace(cuda)
    keep, had = bt.clone(), int(count)
    plan = b200decode.plan_append(sl, bt, free, count, P, new_tokens=nt, max_tokens=T, workspace=ws)
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -9
    assert (plan.slot_mapping == -1).all() and (plan.query_starts == 0).all()
    assert torch.equal(plan.cache_seqlens, sl) and int(plan.free_count) == had and torch.equal(bt, keep)
    # huge counts whose sum passes 32 bits
    nt.fill_(2 ** 31 - 1)
    plan = b200decode.plan_append(sl, bt, free, count, P, new_tokens=nt, max_tokens=T, workspace=ws)
    with pytest.raises(b200decode.B2DError):
        b200decode.check_device_status(ws)
    assert (plan.slot_mapping == -1).all() and torch.equal(bt, keep)


def test_plan_append_negative_entries(cuda):
    """Negative lengths and counts count as 0, a negative page gives slot -1."""
    bt = torch.tensor([[3, 0, 0], [-2, 0, 0], [5, 6, 0]], dtype=torch.int32, device=cuda)
    free = torch.tensor([10, 11, 12, 0], dtype=torch.int32, device=cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    plan = b200decode.plan_append(i32([-7, 2, 8]), bt, free, i32([3]), 4, new_tokens=i32([2, 1, -3]), max_tokens=4)
    assert plan.slot_mapping.tolist() == [48, 49, -1, -1]
    assert plan.query_starts.tolist() == [0, 2, 3, 3]
    assert plan.cache_seqlens.tolist() == [2, 3, 8] and int(plan.free_count) == 2
    assert bt.tolist() == [[12, 0, 0], [-2, 0, 0], [5, 6, 0]]


@pytest.mark.parametrize("B,P,hi,frac", [(1, 16, 50, 1.0), (7, 1, 30, 0.5), (600, 16, 300, 0.1), (2000, 32, 100, 0.9),
                                         (30, 16, 0, 0.5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_pages(cuda, B, P, hi, frac, in_place):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, hi + 1, (B,), generator=g).tolist()
    done = (torch.rand(B, generator=g) < frac).tolist()
    pages = sum((n + P - 1) // P for n in lens) + 4
    bt, free, count = pool_of(B, hi // P + 2, pages, P, lens, 3, cuda)
    want, n = free.tolist(), int(count)
    for b in range(B):
        if done[b]:
            for i in range((lens[b] + P - 1) // P):
                want[n] = int(bt[b, i])
                n += 1
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    fin = torch.tensor(done, device=cuda)
    kw = dict(seqlens_out=sl, free_count_out=count) if in_place else {}
    after, cnt = b200decode.release_pages(sl, bt, fin, free, count, P, **kw)
    assert free.tolist() == want and int(cnt) == n
    assert after.tolist() == [0 if d else L for d, L in zip(done, lens)]


def test_release_that_does_not_fit_changes_nothing(cuda):
    bt, free, count = pool_of(5, 4, 15, 16, [40] * 5, 4, cuda)
    short = free[:10].clone()
    had = short.clone()
    count.fill_(8)
    sl = torch.full((5,), 40, dtype=torch.int32, device=cuda)
    ws = b200decode.DecodeWorkspace(cuda)
    after, cnt = b200decode.release_pages(sl, bt, torch.ones(5, dtype=torch.bool, device=cuda), short, count, 16,
                                          workspace=ws)
    with pytest.raises(b200decode.B2DError) as e:
        b200decode.check_device_status(ws)
    assert e.value.code == -9
    assert torch.equal(after, sl) and int(cnt) == 8 and torch.equal(short, had)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(cuda, kv, captured):
    """A batch on a shared prompt decodes some steps: plan_append ->
    append_kv -> decode_shared_prefix, each step's result against the 64-bit
    reference over everything appended so far; two requests finish, give their
    pages back and start again.  Captured: the step is one CUDA graph."""
    B, P, hkv, hq, d, prompt = 9, 16, 2, 8, 128, 150
    gen = torch.Generator(device=cuda).manual_seed(5)
    npre = (prompt + P - 1) // P
    pages = npre + 24
    ks, vs = (torch.tensor([0.02, 0.05], device=cuda), torch.tensor([0.04, 0.03], device=cuda)) \
        if kv == torch.float8_e4m3fn else (None, None)
    k = torch.zeros(pages, P, hkv, d, dtype=kv, device=cuda)
    v = torch.zeros(pages, P, hkv, d, dtype=kv, device=cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(cuda)
    count = i32([pages])
    # the prompt itself goes through the pool as a request of its own
    pbt = torch.zeros(1, npre, dtype=torch.int32, device=cuda)
    plan = b200decode.plan_append(i32([0]), pbt, free, count, P, new_tokens=i32([prompt]), max_tokens=prompt)
    count = plan.free_count
    pk, pv = (torch.randn(prompt, hkv, d, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    b200decode.append_kv(pk, pv, k, v, plan.slot_mapping, k_scale=ks, v_scale=vs)
    plen = plan.cache_seqlens
    bt = torch.zeros(B, 4, dtype=torch.int32, device=cuda)
    lens = i32([0] * B)
    q = torch.zeros(B, hq, d, dtype=torch.bfloat16, device=cuda)
    key, val = (torch.zeros(B, hkv, d, dtype=torch.bfloat16, device=cuda) for _ in range(2))

    def step():
        plan = b200decode.plan_append(lens, bt, free, count, P, seqlens_out=lens, free_count_out=count)
        b200decode.append_kv(key, val, k, v, plan.slot_mapping, k_scale=ks, v_scale=vs)
        return b200decode.decode_shared_prefix(q, k, v, plen, pbt, lens, bt, k_scale=ks, v_scale=vs)

    graph = None
    if captured:
        state = [x.clone() for x in (lens, count, bt)]
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        for x, s in zip((lens, count, bt), state):
            x.copy_(s)
    for i in range(22):
        for t, n in ((q, hq), (key, hkv), (val, hkv)):
            t.copy_(torch.randn(B, n, d, generator=gen, device=cuda))
        if graph is None:
            result = step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        if i % 7 == 0 or i == 21:
            for b in range(B):
                n = int(lens[b])
                parts = [attend(q[b:b + 1].double(), gather(k, ks, r, m, "NHD"), gather(v, vs, r, m, "NHD"),
                                d ** -0.5, kv) for r, m in ((pbt[0], prompt), (bt[b], n))]
                ref = merge2(*parts)
                check(result[0][b:b + 1], ref[0], ref[2], u_of(torch.bfloat16), f"step {i} out")
                check_lse(result[1][b:b + 1], ref[1], ref[3])
        if i == 9:
            fin = torch.zeros(B, dtype=torch.bool, device=cuda)
            fin[2] = fin[6] = True
            b200decode.release_pages(lens, bt, fin, free, count, P, seqlens_out=lens, free_count_out=count)
    b200decode.check_device_status()
    want = [12 if b in (2, 6) else 22 for b in range(B)]
    assert lens.tolist() == want
    used = sum((n + P - 1) // P for n in want) + npre
    assert int(count) == pages - used
    held = pbt[0].tolist() + [int(bt[b, j]) for b in range(B) for j in range((want[b] + P - 1) // P)]
    assert sorted(held + free[:int(count)].tolist()) == list(range(pages))
