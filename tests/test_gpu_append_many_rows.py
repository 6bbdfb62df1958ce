"""Norm, rotation and the way into the pages for whole prompts: beyond 3552 rows a CTA takes four of them at a time."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [0, 15, 16, 200, 31, 1, 7, 0, 33, 5, 64]
HEAD = [1, 2, 0, 3, 701, 1, 1, 0, 1503, 5]  # (slots begin and end inside four rows, some have none)


def _inputs(T, Hq, heads, dim, dtype, rot, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    qkv = (torch.randn(T, (Hq + 2 * heads) * dim, generator=gen, device="cuda") * 3).to(dtype)
    w = (1 + 0.3 * torch.randn(2, dim, generator=gen, device="cuda")).unbind(0)
    pos = torch.randint(0, 1 << 20, (T,), generator=gen, device="cuda", dtype=torch.int32)
    inv = torch.from_numpy(1e4 ** (-np.arange(0, rot, 2) / max(rot, 1))).cuda()
    return qkv, [x.unflatten(1, (-1, dim)) for x in qkv.split([Hq * dim, heads * dim, heads * dim], dim=1)], w, pos, inv


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,Hq,heads,dtype,layout,T", [
    (64, 64, 8, 1, "bf16", "heads", 3553), (64, 16, 5, 5, "fp16", "tokens", 3554), (64, 0, 3, 2, "bf16", "gap", 3555),
    (128, 128, 7, 2, "bf16", "gap", 3555), (128, 96, 16, 4, "fp16", "heads", 3556), (128, 0, 4, 2, "fp16", "pages", 5001),
    (256, 256, 3, 1, "fp16", "heads", 3553), (256, 64, 8, 2, "bf16", "tokens", 3554), (256, 0, 1, 1, "bf16", "odd", 3555)])  # fmt: skip
def test_rows_of_many_slots(dim, rot, Hq, heads, dtype, layout, T, interleaved):
    import arcinfer_b200 as ab
    import kvutil as kv
    from test_gpu_kvcache import _append64, _near

    dt, behind = kv.DTYPES[dtype], 2
    nodes = HEAD + [T - behind - sum(HEAD)]
    cache, _ = kv.make_cache(dim + rot, LENS, nodes, heads, 16, dim, dt, layers=2, layout=layout)
    off = np.concatenate([[0], np.cumsum(nodes)])
    n = int(off[-1])
    qkv, (q, k, v), w, pos, inv = _inputs(T, Hq, heads, dim, dt, rot, dim + T)
    pos[0], pos[1] = 0, 2**31 - 1
    before = qkv.clone()
    slot = torch.from_numpy(np.repeat(np.arange(len(nodes)), nodes)).cuda()
    place = cache.length[slot].long() + torch.arange(n, device="cuda") - torch.from_numpy(off).cuda()[slot]
    page = cache.table[slot, place // 16].long()
    written = torch.zeros(cache.k.shape[1:4], dtype=torch.bool, device="cuda")
    written[page, :, place % 16] = True
    for weights in (w, (None, w[1]), (None, None)):
        cache.k.fill_(3.0), cache.v.fill_(3.0)
        out = torch.full((T, Hq, dim), 9.0, dtype=dt, device="cuda")
        ab.cache_append(cache, q, k, v, kv.i32(off), pos, inv, layer=1, q_weight=weights[0], k_weight=weights[1], eps=1e-5, interleaved=interleaved, q_out=out)
        torch.cuda.synchronize()
        assert int(cache.status.item()) == 0 and torch.equal(qkv, before)
        _near(out[:n], *_append64(q[:n], weights[0], pos[:n], inv, rot, interleaved, 1e-5), dt)
        assert (out[n:] == 9.0).all()
        wk, size = _append64(k[:n], weights[1], pos[:n], inv, rot, interleaved, 1e-5)
        _near(cache.k[1][page, :, place % 16], wk, size, dt)
        assert torch.equal(cache.v[1][page, :, place % 16], v[:n])
        assert (cache.k[1][~written] == 3.0).all() and (cache.v[1][~written] == 3.0).all() and (cache.k[0] == 3.0).all() and (cache.v[0] == 3.0).all()
    # in place of the queries
    ab.cache_append(cache, q, k, v, kv.i32(off), pos, inv, layer=1, eps=1e-5, interleaved=interleaved, q_out=q)
    torch.cuda.synchronize()
    assert torch.equal(q[:n], out[:n]) and torch.equal(qkv[n:], before[n:]) and torch.equal(qkv[:, Hq * dim :], before[:, Hq * dim :])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_row_outside_the_pages_among_others(dim):
    """its query is written, its key and value are not, and the three rows beside it are as ever"""
    import arcinfer_b200 as ab
    import kvutil as kv

    T, Hq, heads = 4002, 4, 2
    nodes = [1001, 1002, 1999]  # (rows 1000 and 2002 are a slot's last; the fours they are in go on in the next slot)
    cache, _ = kv.make_cache(dim, [0, 5, 3], nodes, heads, 16, dim)
    cache.k.fill_(3.0), cache.v.fill_(3.0)
    # slot 0: the page of its last rows is not there; slot 1: 1007 tokens, room for 992 of them
    cache.table[0, 1000 // 16] = -1
    cache.used[1] -= 1
    off = kv.i32(np.concatenate([[0], np.cumsum(nodes)]))
    _, (q, k, v), w, pos, inv = _inputs(T, Hq, heads, dim, cache.dtype, dim, dim)
    out = ab.cache_append(cache, q, k, v, off, pos, inv, q_weight=w[0], k_weight=w[1])
    torch.cuda.synchronize()
    assert int(cache.status.item()) == 9
    good, _ = kv.make_cache(dim, [0, 5, 3], nodes, heads, 16, dim)
    assert torch.equal(ab.cache_append(good, q, k, v, off, pos, inv, q_weight=w[0], k_weight=w[1]), out)
    torch.cuda.synchronize()
    assert int(good.status.item()) == 0
    lost = set(range(992, 1001)) | set(range(1001 + 992 - 5, 2003))
    slot = np.repeat(np.arange(3), nodes)
    place = good.length.cpu().numpy()[slot] + np.arange(T) - np.concatenate([[0], np.cumsum(nodes)])[slot]
    page, at = torch.from_numpy(good.table.cpu().numpy()[slot, place // 16]).long().cuda(), torch.from_numpy(place % 16).cuda()
    kept = torch.tensor([t not in lost for t in range(T)], device="cuda")
    for a, b in ((cache.k[0], good.k[0]), (cache.v[0], good.v[0])):
        x, y = a[page, :, at], b[page, :, at]
        assert torch.equal(x[kept], y[kept]) and (x[~kept] == 3.0).all()
    assert int((cache.v[0] != 3.0).any(dim=3).sum().item()) == int(kept.sum().item()) * heads
