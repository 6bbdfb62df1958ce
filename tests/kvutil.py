"""A paged cache with known contents for the tests, and the plain implementations they compare with (64 bits)."""
import math

import numpy as np
import torch

import arcinfer_b200 as ab

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a rounding step, relative
# half a step among the subnormal numbers: fp16's begin at 2^-14 with 10 bits behind the point, bf16's at 2^-126 with 7
SMALLEST = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}


def i32(a, device="cuda"):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)


def pool(layers, n_pages, heads, page, dim, dtype, layout, fill=float("nan")):
    """[layers, pages, heads, page, dim] over memory of several orders"""
    if layout == "heads":  # a head's rows of a page side by side
        return torch.full((layers, n_pages, heads, page, dim), fill, dtype=dtype, device="cuda")
    if layout == "tokens":  # a token's heads side by side
        return torch.full((layers, n_pages, page, heads, dim), fill, dtype=dtype, device="cuda").transpose(2, 3)
    if layout == "pages":  # a page's layers side by side
        return torch.full((n_pages, layers, heads, page, dim), fill, dtype=dtype, device="cuda").transpose(0, 1)
    if layout == "odd":  # pages that begin anywhere between two rows
        n = heads * page * dim + 8
        return torch.full((layers, n_pages * n), fill, dtype=dtype, device="cuda").as_strided((layers, n_pages, heads, page, dim), (n_pages * n, n, page * dim, dim, 1))
    # rows with a gap behind them, and pages with one
    wide = torch.full((layers, n_pages, heads * page + 3, dim + 8), fill, dtype=dtype, device="cuda")
    return wide[:, :, : heads * page, :dim].unflatten(2, (heads, page))


def make_cache(seed, lens, rooms, heads=2, page=16, dim=128, dtype=torch.bfloat16, layers=1, layout="heads", spare=5, max_pages=None, scale=1.0):
    """A cache of len(lens) slots; slot s has lens[s] settled tokens and pages for rooms[s] more. Places
    0 .. lens + rooms hold normal numbers, every other row of the pools NaN. Returns the cache and, per
    slot, its keys and values [layers, heads, lens + rooms, dim]."""
    g = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    used = [-(-(n + r) // page) for n, r in zip(lens, rooms)]
    total = sum(used) + spare
    order = g.permutation(total)
    table = np.full((len(lens), max_pages or max(used) + 2), -1)
    k, v = (pool(layers, total, heads, page, dim, dtype, layout) for _ in range(2))
    rows, at = [], 0
    for s, (n, r) in enumerate(zip(lens, rooms)):
        table[s, : used[s]] = order[at : at + used[s]]
        at += used[s]
        pair = []
        for x in (k, v):
            y = (torch.randn(layers, heads, n + r, dim, generator=gen, device="cuda") * scale).to(dtype)
            place = torch.arange(n + r, device="cuda")
            pages = torch.from_numpy(table[s]).cuda()[place // page]
            for layer in range(layers):
                x[layer][pages, :, place % page] = y[layer].transpose(0, 1)
            pair.append(y)
        rows.append(pair)
    ref = np.zeros(total, np.int64)
    for s in range(len(lens)):
        ref[table[s, : used[s]]] += 1
    return ab.KVCache(k, v, i32(table), i32(used), i32(ref), i32(lens)), rows


def random_parents(g, n, back=4):
    return [-1 if i == 0 else max(0, i - 1 - int(g.integers(0, back))) for i in range(n)]


def attention64(q, k, v, length, mask, scale):
    """q [n, Hq, dim], k / v [heads, length + n, dim], mask: n ints. (out, lse, sum of weight * |value|) in
    64 bits over the places a row sees, and over no others."""
    n, Hq, dim = q.shape
    heads = k.shape[0]
    out = torch.zeros(n, Hq, dim, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(n):
        seen = list(range(length)) + [length + j for j in range(n) if (mask[i] >> j) & 1]
        if not seen:
            continue
        kk, vv = (x[:, seen].double().repeat_interleave(Hq // heads, dim=0) for x in (k, v))
        x = torch.einsum("hd,hpd->hp", q[i].double(), kk) * scale
        lse[i] = torch.logsumexp(x, dim=1)
        p = torch.exp(x - lse[i][:, None])
        out[i] = torch.einsum("hp,hpd->hd", p, vv)
        size[i] = torch.einsum("hp,hpd->hd", p, vv.abs())
    return out, lse, size


def check_attention(got, lse, q, cache_rows, lens, off, masks, scale, layer=0):
    """Each value within half a step of the result (its rounding) and half a step of sum weight * |value|
    (each weight is rounded once before the product), and 2^-16 of that sum for all that is done in 32
    bits: 2^-22 a value for the exponential, and scores whose terms add up to at most 2^7 here, 2^-24 each
    in products and sums, 2^-17 in the exponent. Weights among fp16's subnormal numbers are off by 2^-25
    each where the sum of all is at least 2^7: 2^-32 of the largest value a place."""
    u = HALF_STEP[q.dtype]
    for s, n in enumerate(lens):
        a, b = off[s], off[s + 1]
        if a == b:
            continue
        want, wl, size = attention64(q[a:b], cache_rows[s][0][layer], cache_rows[s][1][layer], n, masks[a:b], scale)
        err = (got[a:b].double() - want).abs()
        small = SMALLEST[q.dtype] * (1 + (n + b - a) * 2.0**-7 * cache_rows[s][1][layer].double().abs().max().item())
        bound = u * want.abs() + (u + 2.0**-16) * size + small
        worst = (err / bound).max().item()
        assert not torch.isnan(got[a:b]).any() and worst <= 1.0, (s, n, b - a, worst)
        if lse is not None:
            fin = torch.isfinite(wl)
            assert torch.equal(torch.isfinite(lse[a:b]), fin), (s, n)
            assert ((lse[a:b].double() - wl).abs()[fin] <= 2.0**-16 * (1 + wl.abs()[fin])).all(), (s, n)
