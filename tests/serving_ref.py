"""64-bit reference of ragged attention over paged caches, with an error bound
for each output, and small input makers.

Bound of `out` (elementwise), with A = sum softmax |v| of the row:
  * out is rounded once to its type: u_out |out|, u = eps / 2
  * the softmax weights enter the second product rounded to 16 bits: u_p A
    (bf16 caches: bf16; fp16 and e4m3 caches: fp16, whose subnormal weights
    are off by at most 2^-25 of the largest: L 2^-25 max|v|)
  * a score is off by at most ds = 2^-24 (D + 4) s_abs, s_abs = scale sum |q k|
    (fp32 products and sums), a weight by 2 ds (its own score and the
    maximum), plus 2^-21 for exp2 and the normalisation: (2 ds + 2^-20) A
  * e4m3 caches take q in fp16, whose values under 2^-14 are off by 2^-25:
    part of ds: scale 2^-25 sum |k|
`lse` is off by ds, the errors of exp2, log2 and their scaling (2^-21 (1 +
|lse|)) and of the fp32 sum of L terms (L 2^-24).
"""
from __future__ import annotations

import torch


def gather(cache, scale, row, n, layout):
    """Tokens 0..n of one block-table row, [n, Hkv, D] float64."""
    if layout == "vllm_k":
        c = cache.permute(0, 3, 1, 2, 4).flatten(3)
    elif layout == "vllm_v":
        c = cache.permute(0, 3, 1, 2)
    elif layout == "HND":
        c = cache.permute(0, 2, 1, 3)
    else:
        c = cache
    P = c.shape[1]
    pg = row[: (n + P - 1) // P].long()
    x = c.view(torch.uint8)[pg].view(c.dtype) if c.dtype == torch.float8_e4m3fn else c[pg]
    x = x.double().flatten(0, 1)[:n]
    return x if scale is None else x * scale.double()[None, :, None]


def attend(q, k, v, scale, cache_dtype):
    """q [T, Hq, D], k and v [L, Hkv, D] float64 -> out, lse and their bounds."""
    T, hq, d = q.shape
    L, hkv, _ = k.shape
    u_p = 2.0 ** -8 if cache_dtype == torch.bfloat16 else 2.0 ** -11
    if L == 0:
        z = torch.zeros_like(q)
        return z, torch.full((T, hq), float("-inf"), dtype=q.dtype, device=q.device), z, z[..., 0]
    grp = hq // hkv
    k, v = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
    s = torch.einsum("thd,lhd->thl", q, k) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.softmax(s, -1)
    out = torch.einsum("thl,lhd->thd", p, v)
    ab = torch.einsum("thl,lhd->thd", p, v.abs())
    s_abs = (torch.einsum("thd,lhd->thl", q.abs(), k.abs()) * abs(scale)).amax(-1)
    ds = 2.0 ** -24 * (d + 4) * s_abs
    if cache_dtype == torch.float8_e4m3fn:
        ds = ds + abs(scale) * 2.0 ** -25 * k.abs().sum(-1).amax(0)[None]
    tol = ab * (u_p + 2 * ds[..., None] + 2.0 ** -20)
    if u_p < 2.0 ** -8:
        tol = tol + L * 2.0 ** -25 * v.abs().amax()
    return out, lse, tol, ds + 2.0 ** -21 * (1 + lse.abs()) + L * 2.0 ** -24


def merge2(a, b):
    """Merge two (out, lse, tol, ltol)."""
    lse = torch.logaddexp(a[1], b[1])
    safe = torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)
    w = [torch.exp(x[1] - safe)[..., None] for x in (a, b)]
    dl = (a[3] + b[3])[..., None]
    out = a[0] * w[0] + b[0] * w[1]
    tol = a[2] * w[0] + b[2] * w[1] + (2 * dl + 2.0 ** -20) * (a[0].abs() * w[0] + b[0].abs() * w[1])
    return out, lse, tol, torch.maximum(a[3], b[3]) + 2.0 ** -21 * (1 + safe.abs())


def check(got, ref, tol, u_out, what):
    g = got.double()
    assert torch.isfinite(g).all(), f"{what}: not finite"
    # Rounding to the output type: half a step, eps / 2 of the value, but never
    # less than half the type's smallest step (fp16: values under 2^-14 are
    # multiples of 2^-24, so off by up to 2^-25 whatever their size).
    least = torch.finfo(got.dtype).smallest_normal * u_out
    bad = (g - ref).abs() - (tol + (u_out * (ref.abs() + tol)).clamp(min=least))
    assert bad.max().item() <= 0, f"{what}: {bad.max().item():.3e} over the bound, at {int(bad.argmax())}"


def check_lse(got, ref, tol):
    g = got.double()
    assert torch.equal(torch.isneginf(g), torch.isneginf(ref)), "lse -inf pattern differs"
    fin = torch.isfinite(ref)
    assert torch.isfinite(g[fin]).all(), "lse not finite"
    over = (g - ref).abs()[fin] - tol[fin]
    assert over.numel() == 0 or over.max().item() <= 0, f"lse: {over.max().item():.3e} over the bound"


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def tables(lens, P, perm, at, width=None):
    need = [(int(n) + P - 1) // P for n in lens]
    width = width or max([1] + need)
    bt = torch.zeros(len(need), width, dtype=torch.int32)
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, at


def caches(gen, device, pages, P, hkv, d, kv, layout):
    """K and V caches in any layout, values N(0, 1) (e4m3: after their scales);
    scales of e4m3 caches."""
    shape = {"NHD": (pages, P, hkv, d), "HND": (pages, hkv, P, d), "vllm": (pages, P, hkv, d)}[layout]
    ks = vs = None
    if kv == torch.float8_e4m3fn:
        ks, vs = (0.02 + 0.1 * torch.rand(hkv, generator=gen, device=device) for _ in range(2))
    out = []
    for sc in (ks, vs):
        x = torch.randn(shape, generator=gen, device=device)
        if sc is not None:
            x = (x / (sc[None, :, None, None] if layout == "HND" else sc[None, None, :, None])).clamp(-448, 448)
        out.append(x.to(kv))
    k, v = out
    if layout == "vllm":
        x = 8
        k = k.reshape(pages, P, hkv, d // x, x).permute(0, 2, 3, 1, 4).contiguous()
        v = v.permute(0, 2, 3, 1).contiguous()
    return k, v, ks, vs
