"""The serving operators that stand beside paged decode and KV append, as cases to be measured.

Operators: decode over a prefix that groups of sequences share (`shared`), cross attention of
ragged query tokens to paged encoder states (`cross`), the block tables and slot map of the next
append (`append`), the release of finished requests' pages (`release`), and the merge of attention
states over disjoint parts of the keys (`merge`).

`own` selects between the plain forms below (elementary torch operations in 32 bits) and the
framework's calls.
"""
import math

import torch

own = False

if torch.cuda.is_available():
    DEV = torch.device("cuda", 0)
else:
    DEV = torch.device("cpu")

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp8": 1, "fp32": 4}


def _api():
    import os
    import sys
    pkg = os.path.join(os.getcwd(), "roofline-analysis_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import b200decode
    return b200decode


# ----------------------------------------------------------------------------- cases

def listed():
    return [
        # Four chat requests on one system prompt, a few turns in: the latency of one decode step.
        dict(name="shared_small", op="shared", q="bf16", kv="bf16", B=4, Hq=32, Hkv=8, D=128, P=16,
             groups=1, prefix_lo=1024, prefix_hi=1024, own_lo=16, own_hi=256),
        # A full decode batch on a long tool-and-instructions prompt, FP8 cache.
        dict(name="shared_fp8_batch", op="shared", q="bf16", kv="fp8", B=256, Hq=32, Hkv=8, D=128, P=16,
             groups=1, prefix_lo=8191, prefix_hi=8191, own_lo=64, own_hi=1024),
        # Requests over seven documents of different length, several questions to each.
        dict(name="shared_documents", op="shared", q="bf16", kv="bf16", B=67, Hq=64, Hkv=8, D=128, P=64,
             groups=7, prefix_lo=1000, prefix_hi=30000, own_lo=1, own_hi=700),
        # The largest: parallel samples of one 128k-token context.
        dict(name="shared_long", op="shared", q="bf16", kv="bf16", B=64, Hq=64, Hkv=8, D=128, P=64,
             groups=1, prefix_lo=131072, prefix_hi=131072, own_lo=200, own_hi=2000),
        # A speech decoder's first tokens against one utterance's states.
        dict(name="cross_small", op="cross", q="fp16", kv="fp16", B=2, Hq=16, Hkv=16, D=64, P=16,
             t_lo=3, t_hi=5, k_lo=300, k_hi=700),
        # A translation batch: ragged targets against ragged sources.
        dict(name="cross_ragged", op="cross", q="bf16", kv="bf16", B=48, Hq=16, Hkv=16, D=64, P=16,
             t_lo=1, t_hi=200, k_lo=1, k_hi=1500),
        # Long text against image or audio states, grouped heads.
        dict(name="cross_large", op="cross", q="bf16", kv="bf16", B=16, Hq=32, Hkv=8, D=128, P=64,
             t_lo=256, t_hi=1024, k_lo=2048, k_hi=6500),
        # One new token for each request of a decode batch.
        dict(name="append_decode", op="append", B=256, P=16, len_lo=0, len_hi=8192, new_lo=1, new_hi=1),
        # A large mixed step: prompt chunks and single tokens.
        dict(name="append_prompts", op="append", B=1000, P=16, len_lo=0, len_hi=3000, new_lo=0, new_hi=600),
        # The requests that finished in a step give their pages back.
        dict(name="release_step", op="release", B=512, P=16, len_lo=0, len_hi=8192, done=0.1),
        # Eight ranks' states of a context-parallel decode.
        dict(name="merge_ranks", op="merge", dtype="bf16", out="bf16", N=8, B=256, H=32, D=128, empty=0.1),
        # Two states of 32-bit partial results, small batch.
        dict(name="merge_pair", op="merge", dtype="fp32", out="bf16", N=2, B=7, H=64, D=128, empty=0.2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "shared", "cross", "cross", "cross", "append", "release", "merge"])
    if op == "shared":
        kv = rng.choice(["bf16", "fp8", "fp16"])
        hkv = rng.choice([1, 2, 4, 8])
        grp = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        d = rng.choice([64, 128, 128])
        p = rng.choice([16, 32, 48, 64, 128])
        b = _log(rng, 2, 300)
        groups = min(b, rng.choice([1, 1, 2, 5, 11]))
        own = _log(rng, 2, 2000)
        # tokens x query heads of the prefix stay below the largest listed case's
        top = min(131072, max(64, 64 * 64 * 131072 // (4 * b * hkv * grp)))
        top = min(top, 400000 // groups)
        hi = _log(rng, 33, max(64, top))
        return dict(op=op, q="fp16" if kv == "fp16" else "bf16", kv=kv, B=b, Hq=hkv * grp, Hkv=hkv, D=d, P=p,
                    groups=groups, prefix_lo=max(1, hi // 2), prefix_hi=hi,
                    own_lo=max(0, own // 8), own_hi=min(own, 4000000 // (b * hkv)))
    if op == "cross":
        kv = rng.choice(["bf16", "fp8", "fp16"])
        hkv = rng.choice([1, 4, 8, 16])
        grp = rng.choice([1, 1, 2, 4, 6])
        b = _log(rng, 1, 64)
        t = _log(rng, 2, 1024 if b <= 16 else 200)
        k = _log(rng, 5, 6500 if b <= 16 else 3500)
        k = max(5, min(k, 16 * 8 * 6500 // (b * hkv)))
        t = max(2, min(t, 16 * 32 * 1024 * 6500 // (b * hkv * grp * k)))
        return dict(op=op, q="fp16" if kv == "fp16" else "bf16", kv=kv, B=b, Hq=hkv * grp, Hkv=hkv,
                    D=rng.choice([64, 128]), P=rng.choice([16, 32, 64, 80, 128]),
                    t_lo=rng.choice([0, 1, max(1, t // 2)]), t_hi=t, k_lo=rng.choice([1, max(1, k // 3)]), k_hi=k)
    if op == "append":
        b = _log(rng, 1, 4000)
        new = rng.choice([1, 1, _log(rng, 2, max(3, 600000 // b))])
        return dict(op=op, B=b, P=rng.choice([1, 5, 16, 32, 64, 128]), len_lo=0,
                    len_hi=_log(rng, 10, max(20, min(30000, 4000000 // b))),
                    new_lo=1 if new == 1 else 0, new_hi=new)
    if op == "release":
        b = _log(rng, 1, 4000)
        return dict(op=op, B=b, P=rng.choice([1, 5, 16, 32, 64, 128]), len_lo=0,
                    len_hi=_log(rng, 10, max(20, min(30000, 4000000 // b))), done=round(rng.uniform(0.02, 1.0), 3))
    dt = rng.choice(["bf16", "fp16", "fp32"])
    return dict(op=op, dtype=dt, out=dt if dt != "fp32" else rng.choice(["fp32", "bf16", "fp16"]),
                N=rng.choice([1, 2, 3, 4, 8, 13]), B=_log(rng, 1, 500), H=rng.choice([1, 6, 8, 32, 40, 64]),
                D=rng.choice([64, 128, 192, 256, 512]), empty=rng.choice([0.0, 0.1, 0.5]))


# ----------------------------------------------------------------------------- inputs

def _lens(gen, n, lo, hi):
    """n lengths spread evenly over [lo, hi], in random order (their sum is the case's own)."""
    x = torch.linspace(lo, hi, n, dtype=torch.float64).round().long() if n > 1 else torch.tensor([hi])
    return x[torch.randperm(n, generator=gen)]


def _table(lens, P, pool, at, width=None):
    """Block table of `lens` tokens each, pages from pool[at:]; rows padded with page 0."""
    pages = (lens + P - 1) // P
    width = max(1, int(pages.max()) if len(lens) else 1) if width is None else width
    first = torch.cumsum(pages, 0) - pages + at
    col = torch.arange(width)
    idx = first[:, None] + col[None]
    used = col[None] < pages[:, None]
    bt = torch.where(used, pool[idx.clamp(max=len(pool) - 1)], torch.zeros((), dtype=pool.dtype))
    return bt.to(torch.int32), at + int(pages.sum())


def _caches(case, pages, gen):
    hkv, d, P = case["Hkv"], case["D"], case["P"]
    dt = _DT[case["kv"]]
    shape = (pages, P, hkv, d)
    ks = vs = None
    if case["kv"] == "fp8":
        # values after per-head quantisation: scales as a calibrated cache has them
        ks = 0.01 + 0.09 * torch.rand(hkv, generator=gen, device=DEV)
        vs = 0.01 + 0.09 * torch.rand(hkv, generator=gen, device=DEV)
    out = []
    for sc in (ks, vs):
        c = torch.empty(shape, dtype=dt, device=DEV)
        step = max(1, (1 << 27) // (P * hkv * d))
        for i in range(0, pages, step):
            x = torch.randn((min(pages, i + step) - i,) + shape[1:], generator=gen, device=DEV)
            if sc is not None:
                x = (x / sc[:, None]).clamp_(-448.0, 448.0)
            c[i:i + step] = x.to(dt)
        out.append(c)
    return out[0], out[1], ks, vs


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed * 1000003 + 17)
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 29)
    op = case["op"]
    s = dict(op=op, case=case)
    if op == "shared":
        B, P, G = case["B"], case["P"], case["groups"]
        plen = _lens(host, G, case["prefix_lo"], case["prefix_hi"])
        olen = _lens(host, B, case["own_lo"], max(case["own_lo"], case["own_hi"]))
        # groups of random sizes, each at least one sequence
        cuts = torch.randperm(B - 1, generator=host)[:G - 1].sort().values + 1 if G > 1 else torch.zeros(0, dtype=torch.int64)
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([B])])
        pages = int(((plen + P - 1) // P).sum() + ((olen + P - 1) // P).sum())
        pool = torch.randperm(max(1, pages), generator=host)
        pbt, at = _table(plen, P, pool, 0)
        bt, _ = _table(olen, P, pool, at)
        kc, vc, ks, vs = _caches(case, max(1, pages), gen)
        q = torch.randn(B, case["Hq"], case["D"], generator=gen, device=DEV).to(_DT[case["q"]])
        s.update(q=q, kc=kc, vc=vc, ks=ks, vs=vs, plen=plen.to(torch.int32).to(DEV), pbt=pbt.to(DEV),
                 olen=olen.to(torch.int32).to(DEV), bt=bt.to(DEV), starts=starts.to(torch.int32).to(DEV),
                 most=int((starts[1:] - starts[:-1]).max()), scale=case["D"] ** -0.5)
    elif op == "cross":
        B, P = case["B"], case["P"]
        tq = _lens(host, B, case["t_lo"], max(case["t_lo"], case["t_hi"]))
        kl = _lens(host, B, case["k_lo"], max(case["k_lo"], case["k_hi"]))
        pages = int(((kl + P - 1) // P).sum())
        bt, _ = _table(kl, P, torch.randperm(pages, generator=host), 0)
        kc, vc, ks, vs = _caches(case, pages, gen)
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(tq, 0)])
        q = torch.randn(int(starts[-1]), case["Hq"], case["D"], generator=gen, device=DEV).to(_DT[case["q"]])
        s.update(q=q, kc=kc, vc=vc, ks=ks, vs=vs, klen=kl.to(torch.int32).to(DEV), bt=bt.to(DEV),
                 starts=starts.to(torch.int32).to(DEV), most=int(tq.max()), scale=case["D"] ** -0.5)
    elif op in ("append", "release"):
        B, P = case["B"], case["P"]
        ln = _lens(host, B, case["len_lo"], case["len_hi"])
        have = (ln + P - 1) // P
        if op == "append":
            new = _lens(host, B, case["new_lo"], case["new_hi"])
            need = (ln + new + P - 1) // P - have
            most = int(((new + P - 1) // P + 1).sum())
            s["new"] = new.to(torch.int32).to(DEV) if case["new_hi"] > 1 else None
            s["tokens"] = int(new.sum())
        else:
            most = 0
            s["done"] = (torch.rand(B, generator=host) < case["done"]).to(DEV)
        # a pool with a few pages more than the step can need, and a table of the longest request's width
        pool = torch.randperm(int(have.sum()) + most + 37, generator=host)
        width = (case["len_hi"] + case.get("new_hi", 0)) // P + 3
        bt, at = _table(ln, P, pool, 0, width)
        free = torch.zeros(len(pool), dtype=torch.int32)
        free[:len(pool) - at] = pool[at:].to(torch.int32)
        s.update(len=ln.to(torch.int32).to(DEV), bt=bt.to(DEV), free=free.to(DEV),
                 count=torch.tensor([len(pool) - at], dtype=torch.int32, device=DEV), P=P)
    else:
        N, B, H, D = case["N"], case["B"], case["H"], case["D"]
        o = torch.randn(N, B, H, D, generator=gen, device=DEV).to(_DT[case["dtype"]])
        l = 8.0 + 1.5 * torch.randn(N, B, H, generator=gen, device=DEV)
        gone = torch.rand(N, B, H, generator=gen, device=DEV) < case["empty"]
        o = o.masked_fill(gone[..., None], 0.0)   # an empty part's state: out 0, lse -inf
        s.update(o=o, l=l.masked_fill(gone, float("-inf")))
    return s


# ----------------------------------------------------------------------------- plain forms

def _gather(cache, scale, bt):
    """Pages bt [R, W] of a cache as [R, W * P, Hkv, D] in 32 bits."""
    x = cache.view(torch.uint8).index_select(0, bt.reshape(-1).long()).view(cache.dtype) \
        if cache.dtype == torch.float8_e4m3fn else cache.index_select(0, bt.reshape(-1).long())
    x = x.float()
    if scale is not None:
        x = x * scale[:, None]
    return x.reshape(bt.shape[0], -1, cache.shape[2], cache.shape[3])


def _attend(q, k, v, lens, scale):
    """q [R, T, Hq, D], k and v [R, L, Hkv, D] (32 bits), lens [R]: unnormalised sums [R, T, Hq, D],
    maxima and sums of the exponentials [R, T, Hq]."""
    R, T, Hq, D = q.shape
    Hkv = k.shape[2]
    grp = Hq // Hkv
    qq = q.float().reshape(R, T, Hkv, grp, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, T * grp, D)
    sc = torch.matmul(qq, k.permute(0, 2, 3, 1)) * scale
    out_of = torch.arange(k.shape[1], device=q.device)[None] >= lens[:, None]
    sc.masked_fill_(out_of[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m0 = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(sc.sub_(m0))
    back = lambda x: x.reshape(R, Hkv, T, grp, -1).permute(0, 2, 1, 3, 4).reshape(R, T, Hq, -1)  # noqa: E731
    return back(torch.matmul(p, v.permute(0, 2, 1, 3))), back(m)[..., 0], back(p.sum(-1, keepdim=True))[..., 0]


def _packed(q, starts, most):
    """Ragged rows q [T, ...] as [G, most, ...], and the place of each row there."""
    n = starts.long()
    idx = n[:-1, None] + torch.arange(most, device=q.device)[None]
    qp = q.index_select(0, idx.clamp(max=q.shape[0] - 1).reshape(-1)).reshape((len(n) - 1, most) + q.shape[1:])
    row = torch.arange(q.shape[0], device=q.device)
    g = torch.searchsorted(n[1:].contiguous(), row, right=True)
    return qp, g * most + (row - n[g])


def _plain_shared(s):
    q = s["q"]
    qp, at = _packed(q, s["starts"], s["most"])
    o1, m1, l1 = _attend(qp, _gather(s["kc"], s["ks"], s["pbt"]), _gather(s["vc"], s["vs"], s["pbt"]), s["plen"], s["scale"])
    o1, m1, l1 = (x.flatten(0, 1).index_select(0, at) for x in (o1, m1, l1))
    o2, m2, l2 = _attend(q[:, None], _gather(s["kc"], s["ks"], s["bt"]), _gather(s["vc"], s["vs"], s["bt"]), s["olen"], s["scale"])
    o2, m2, l2 = o2[:, 0], m2[:, 0], l2[:, 0]
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    l = l1 * w1 + l2 * w2
    out = (o1 * w1[..., None] + o2 * w2[..., None]) / l[..., None]
    return out.to(q.dtype), m + torch.log(l)


def _plain_cross(s):
    q = s["q"]
    qp, at = _packed(q, s["starts"], s["most"])
    o, m, l = _attend(qp, _gather(s["kc"], s["ks"], s["bt"]), _gather(s["vc"], s["vs"], s["bt"]), s["klen"], s["scale"])
    o, m, l = (x.flatten(0, 1).index_select(0, at) for x in (o, m, l))
    return (o / l[..., None]).to(q.dtype), m + torch.log(l)


def _plain_append(s):
    P, bt = s["P"], s["bt"]
    ln = s["len"].long()
    new = s["new"].long() if s["new"] is not None else torch.ones_like(ln)
    have = (ln + P - 1) // P
    need = (ln + new + P - 1) // P - have
    at = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    k = torch.arange(bt.shape[1], device=bt.device)[None] - have[:, None]
    src = s["count"].long() - 1 - (at[:, None] + k)
    fresh = s["free"][src.clamp(0, len(s["free"]) - 1)]
    bt.copy_(torch.where((k >= 0) & (k < need[:, None]), fresh, bt))
    t = torch.arange(s["tokens"], device=bt.device)
    b = torch.searchsorted(ends, t, right=True)
    pos = ln[b] + t - (ends - new)[b]
    slots = bt[b, pos // P].long() * P + pos % P
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    return slots, starts, (ln + new).to(torch.int32), (s["count"] - need.sum()).to(torch.int32), bt


def _plain_release(s):
    P, bt, free = s["P"], s["bt"], s["free"]
    ln = s["len"].long()
    pages = torch.where(s["done"], (ln + P - 1) // P, torch.zeros_like(ln))
    at = torch.cumsum(pages, 0) - pages
    k = torch.arange(bt.shape[1], device=bt.device)[None]
    given = k < pages[:, None]
    free.index_copy_(0, (s["count"].long() + at[:, None] + k)[given], bt[given])
    return torch.where(s["done"], torch.zeros_like(s["len"]), s["len"]), (s["count"] + pages.sum()).to(torch.int32), free


def _plain_merge(s):
    o, l = s["o"].float(), s["l"]
    m = l.amax(0)
    m0 = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    w = torch.exp(l - m0)
    t = w.sum(0)
    out = (o * w[..., None]).sum(0) / torch.where(t == 0, torch.ones_like(t), t)[..., None]
    return out.to(_DT[s["case"]["out"]]), m0 + torch.log(t)


_PLAIN = dict(shared=_plain_shared, cross=_plain_cross, append=_plain_append, release=_plain_release, merge=_plain_merge)


# ----------------------------------------------------------------------------- the framework's calls

def _own(s):
    b2 = _api()
    op = s["op"]
    if op == "shared":
        return b2.decode_shared_prefix(s["q"], s["kc"], s["vc"], s["plen"], s["pbt"], s["olen"], s["bt"], s["scale"],
                                       group_starts=s["starts"], k_scale=s["ks"], v_scale=s["vs"])
    if op == "cross":
        return b2.cross_attention(s["q"], s["kc"], s["vc"], s["klen"], s["bt"], s["scale"], query_starts=s["starts"],
                                  k_scale=s["ks"], v_scale=s["vs"])
    if op == "append":
        plan = b2.plan_append(s["len"], s["bt"], s["free"], s["count"], s["P"], new_tokens=s["new"], max_tokens=s["tokens"])
        return plan.slot_mapping, plan.query_starts, plan.cache_seqlens, plan.free_count, s["bt"]
    if op == "release":
        lens, count = b2.release_pages(s["len"], s["bt"], s["done"], s["free"], s["count"], s["P"])
        return lens, count, s["free"]
    out = torch.empty(s["o"].shape[1:], dtype=_DT[s["case"]["out"]], device=s["o"].device)
    return b2.merge_states(s["o"], s["l"], out=out)


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "shared":
        es, hd = _ES[case["kv"]], case["Hkv"] * case["D"]
        pre = case["groups"] * (case["prefix_lo"] + case["prefix_hi"]) / 2
        mine = case["B"] * (case["own_lo"] + max(case["own_lo"], case["own_hi"])) / 2
        rows = case["B"] * case["Hq"]
        entries = (pre + mine) / case["P"] + 2 * case["B"] + 2 * case["groups"]
        return {"bytes": 2 * es * hd * (pre + mine) + rows * (4 * case["D"] + 4) + 4 * entries,
                "flops": 4 * case["D"] * case["Hq"] * (case["B"] * pre / case["groups"] + mine)}
    if op == "cross":
        es, hd = _ES[case["kv"]], case["Hkv"] * case["D"]
        k = (case["k_lo"] + max(case["k_lo"], case["k_hi"])) / 2
        t = (case["t_lo"] + max(case["t_lo"], case["t_hi"])) / 2
        rows = case["B"] * t * case["Hq"]
        return {"bytes": 2 * es * hd * case["B"] * k + rows * (4 * case["D"] + 4) + 4 * case["B"] * (k / case["P"] + 2),
                "flops": 4 * case["D"] * rows * k}
    if op == "append":
        new = (case["new_lo"] + case["new_hi"]) / 2
        pages = case["B"] * new / case["P"]
        # lengths in and out, token starts, a table entry for each request, new pages read and written, slots
        return {"bytes": 4 * case["B"] * (4 if case["new_hi"] == 1 else 5) + 8 * pages + 8 * case["B"] * new, "flops": 0}
    if op == "release":
        pages = case["done"] * case["B"] * (case["len_lo"] + case["len_hi"]) / 2 / case["P"]
        return {"bytes": 9 * case["B"] + 8 * pages, "flops": 0}
    rows = case["B"] * case["H"]
    return {"bytes": rows * case["N"] * (case["D"] * _ES[case["dtype"]] + 4) + rows * (case["D"] * _ES[case["out"]] + 4),
            "flops": 2 * rows * case["N"] * case["D"]}


# ----------------------------------------------------------------------------- the definition in 64 bits

def _tokens(cache, scale, row, n, P):
    """Tokens 0..n of a block-table row as [n, Hkv, D] in 64 bits."""
    pg = row[: (n + P - 1) // P].long()
    raw = cache.view(torch.uint8)[pg].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[pg]
    x = raw.double().flatten(0, 1)[:n]
    return x if scale is None else x * scale.double()[None, :, None]


def _softmax_over(q, k, v, scale):
    """q [T, Hq, D] against k, v [L, Hkv, D], all in 64 bits: (out, lse)."""
    rep = q.shape[1] // k.shape[1]
    outs, lses = [], []
    for h in range(k.shape[1]):
        qh = q[:, h * rep:(h + 1) * rep].reshape(-1, q.shape[2])
        sc = (qh @ k[:, h].T) * scale
        lse = torch.logsumexp(sc, 1)
        outs.append((torch.softmax(sc, 1) @ v[:, h]).reshape(-1, rep, q.shape[2]))
        lses.append(lse.reshape(-1, rep))
    return torch.cat(outs, 1), torch.cat(lses, 1)


def exact(case, seed):
    op = case["op"]
    if op in ("append", "release"):
        return None   # whole numbers
    s = prepare(case, seed)
    P = case.get("P")
    if op == "merge":
        o, l = s["o"].double(), s["l"].double()
        lse = torch.logsumexp(l, 0)
        w = torch.exp(l - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
        return torch.einsum("nbh,nbhd->bhd", w, o), lse
    q = s["q"].double()
    starts = s["starts"].tolist()
    outs, lses = [], []
    if op == "cross":
        for b, n in enumerate(s["klen"].tolist()):
            if starts[b + 1] > starts[b]:
                k, v = _tokens(s["kc"], s["ks"], s["bt"][b], n, P), _tokens(s["vc"], s["vs"], s["bt"][b], n, P)
                o, l = _softmax_over(q[starts[b]:starts[b + 1]], k, v, s["scale"])
                outs.append(o)
                lses.append(l)
        return torch.cat(outs), torch.cat(lses)
    own_n = s["olen"].tolist()
    for g, n in enumerate(s["plen"].tolist()):
        kp, vp = _tokens(s["kc"], s["ks"], s["pbt"][g], n, P), _tokens(s["vc"], s["vs"], s["pbt"][g], n, P)
        # the prefix's part for all of the group's sequences at once, then each sequence's own part
        op_, lp = _softmax_over(q[starts[g]:starts[g + 1]], kp, vp, s["scale"])
        for i, b in enumerate(range(starts[g], starts[g + 1])):
            if own_n[b] == 0:
                outs.append(op_[i:i + 1])
                lses.append(lp[i:i + 1])
                continue
            ko, vo = _tokens(s["kc"], s["ks"], s["bt"][b], own_n[b], P), _tokens(s["vc"], s["vs"], s["bt"][b], own_n[b], P)
            oo, lo = _softmax_over(q[b:b + 1], ko, vo, s["scale"])
            lse = torch.logaddexp(lp[i:i + 1], lo)
            outs.append(op_[i:i + 1] * torch.exp(lp[i:i + 1] - lse)[..., None] + oo * torch.exp(lo - lse)[..., None])
            lses.append(lse)
    return torch.cat(outs), torch.cat(lses)
