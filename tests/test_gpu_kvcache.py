"""Pages of a cache: reserved, forked, freed, compacted, and written by norm and rotation, against plain restatements."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Plain:
    """the lists of a cache in numpy, with the rules of include/arcsample.h"""

    def __init__(self, cache, page):
        self.page = page
        self.table, self.used, self.ref, self.len = (x.cpu().numpy().copy() for x in (cache.table, cache.used, cache.ref, cache.length))
        self.k, self.v = cache.k.clone(), cache.v.clone()

    def take(self, s, n, at):
        free = np.flatnonzero(self.ref == 0)
        if len(free) < n:
            return False
        self.table[s, at : at + n] = free[:n]
        self.ref[free[:n]] = 1
        return True

    def reserve(self, extra):
        full = False
        for s, e in enumerate(extra):
            if e <= 0:
                continue
            want = -(-(int(self.len[s]) + int(e)) // self.page)
            need = want - int(self.used[s])
            if want > self.table.shape[1]:
                full = True
            elif need > 0 and (full_now := getattr(self, "_out", False)):
                full = full or full_now
            elif need > 0:
                if self.take(s, need, int(self.used[s])):
                    self.used[s] = want
                else:
                    self._out = full = True
        self._out = False
        return full

    def free(self, which):
        for s, w in enumerate(which):
            if w:
                np.subtract.at(self.ref, self.table[s, : self.used[s]], 1)
                self.table[s, : self.used[s]] = -1
                self.used[s] = self.len[s] = 0

    def fork(self, parent):
        done = []
        for s, p in enumerate(parent):
            full, rest = divmod(int(self.len[p]), self.page)
            if p < 0 or self.used[s] or p == s or parent[p] >= 0 or (rest and not self.take(s, 1, full)):
                done.append(0)
                continue
            self.table[s, :full] = self.table[p, :full]
            np.add.at(self.ref, self.table[p, :full], 1)
            if rest:
                a, b = self.table[p, full], self.table[s, full]
                self.k[:, b, :, :rest], self.v[:, b, :, :rest] = self.k[:, a, :, :rest].clone(), self.v[:, a, :, :rest].clone()
            self.used[s], self.len[s] = full + (rest > 0), self.len[p]
            done.append(1)
        return done

    def compact(self, kept, path):
        for s, n in enumerate(kept):
            length = int(self.len[s])
            where = lambda p: (int(self.table[s, p // self.page]), p % self.page)  # noqa: E731
            for x in (self.k, self.v):
                rows = [x[:, where(length + int(j))[0], :, where(length + int(j))[1]].clone() for j in path[s][:n]]
                for i, r in enumerate(rows):
                    pg, t = where(length + i)
                    x[:, pg, :, t] = r
            self.len[s] = length + n
            left = -(-int(self.len[s]) // self.page)
            if left < self.used[s]:
                np.subtract.at(self.ref, self.table[s, left : self.used[s]], 1)
                self.table[s, left : self.used[s]] = -1
                self.used[s] = left

    def check(self, cache, status=0):
        torch.cuda.synchronize()
        assert int(cache.status.item()) == status
        for name, mine, got in (("used", self.used, cache.used), ("ref", self.ref, cache.ref), ("length", self.len, cache.length)):
            assert np.array_equal(mine, got.cpu().numpy()), name
        t = cache.table.cpu().numpy()
        for s, n in enumerate(self.used):
            assert np.array_equal(self.table[s, :n], t[s, :n]), s
        held = torch.from_numpy(np.flatnonzero(self.ref > 0)).cuda()
        for mine, got in ((self.k, cache.k), (self.v, cache.v)):
            bits = lambda x: x[:, held].contiguous().view(torch.int16)  # noqa: E731
            assert torch.equal(bits(mine), bits(got))


@pytest.mark.parametrize("layout", ["heads", "tokens", "pages", "gap"])
@pytest.mark.parametrize("page,dim,dtype", [(16, 64, "bf16"), (32, 128, "fp16"), (256, 256, "bf16")])
def test_a_life_of_many_steps(page, dim, dtype, layout):
    """random calls of all four kinds in a row"""
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(page + dim)
    S = 9
    cache, _ = kv.make_cache(page, [0, 3, page, page + 1, 5 * page - 1, 0, 70, 0, 0], [0] * S, heads=3, page=page, dim=dim, dtype=kv.DTYPES[dtype], layers=2, layout=layout, spare=40,
                             max_pages=40)
    plain = Plain(cache, page)
    for step in range(12):
        extra = [int(x) for x in g.integers(-2, 40, S)]
        ab.cache_reserve(cache, kv.i32(extra))
        assert not plain.reserve(extra)
        plain.check(cache)
        kept, path = np.zeros(S, np.int64), np.full((S, 40), -1)
        for s in range(S):
            room = int(plain.used[s]) * page - int(plain.len[s])
            n = min(room, 40)
            kept[s] = int(g.integers(0, min(n, 11) + 1))
            path[s, : kept[s]] = np.sort(g.permutation(n)[: kept[s]])
        if step % 3 == 0:
            path[:, :5] = np.arange(5)  # whole stretches that stay where they are
            kept = np.minimum(kept, 5)
            kept[plain.used * page - plain.len < 5] = 0
        if step % 2:
            ab.cache_compact(cache, kv.i32(kept), kv.i32(path))
        else:
            out = torch.full((S,), -7, dtype=torch.int32, device="cuda")
            before = cache.length.clone()
            assert ab.cache_compact(cache, kv.i32(kept), kv.i32(path), length_out=out) is out
            assert torch.equal(cache.length, before)
            cache.length.copy_(out)
        plain.compact(kept, path)
        plain.check(cache)
        which = (g.random(S) < 0.3).astype(np.int64)
        ab.cache_free(cache, kv.i32(which))
        plain.free(which)
        plain.check(cache)
        empty, there = np.flatnonzero(plain.used == 0), np.flatnonzero(plain.used > 0)
        parent = np.full(S, -1)
        if len(there):
            for s in empty:
                if g.random() < 0.6:
                    parent[s] = g.choice(there)
        done = ab.cache_fork(cache, kv.i32(parent))
        assert np.array_equal(done.cpu().numpy(), plain.fork(parent))
        plain.check(cache)


def test_many_slots_and_pages():
    """the largest number of slots; more pages than one walk over them takes in; the free ones scattered"""
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(1)
    S, P, page = 4096, 30011, 16
    z = torch.zeros(1, P, 1, page, 64, dtype=torch.bfloat16, device="cuda")
    ref = (g.random(P) < 0.7).astype(np.int64)
    cache = ab.KVCache(z, z.clone(), kv.i32(np.full((S, 4), -1)), kv.i32(np.zeros(S)), kv.i32(ref), kv.i32(np.zeros(S)))
    plain = Plain(cache, page)
    for lo, hi in ((0, 17), (0, 65), (30, 60)):
        extra = g.integers(lo, hi, S)
        ab.cache_reserve(cache, kv.i32(extra))
        full = plain.reserve(extra)
        torch.cuda.synchronize()
        plain.check(cache, 10 if full else 0)
        cache.status.zero_()


@pytest.mark.parametrize("spare", [0, 1, 5, 6, 7])
def test_pages_run_out(spare):
    """all of a slot's pages or none; from the first slot on that goes without, none"""
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, _ = kv.make_cache(3, [10, 16, 0, 40, 7], [0] * 5, page=16, spare=spare, max_pages=6)
    plain = Plain(cache, 16)
    extra = [20, 0, 33, 200, 10]  # 1 page, none, 3 pages, more than a list holds, 1 page
    ab.cache_reserve(cache, kv.i32(extra))
    assert plain.reserve(extra)
    assert [int(x) for x in cache.used.cpu()] == [2 if spare >= 1 else 1, 1, 3 if spare >= 4 else 0, 3, 2 if spare >= 5 else 1]
    plain.check(cache, 10)


def test_more_pages_asked_for_than_an_int_counts():
    import arcinfer_b200 as ab
    import kvutil as kv

    S, most, P = 200, 1 << 24, 50  # 200 x 2^24 pages
    z = torch.zeros(1, P, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    cache = ab.KVCache(z, z.clone(), torch.empty(S, most, dtype=torch.int32, device="cuda"), kv.i32(np.zeros(S)), kv.i32(np.zeros(P)), kv.i32(np.zeros(S)))
    extra = np.full(S, 2**28)
    extra[:2] = 20, 40
    ab.cache_reserve(cache, kv.i32(extra))
    torch.cuda.synchronize()
    assert int(cache.status.item()) == 10 and cache.used.tolist() == [2, 3] + [0] * (S - 2)
    assert cache.table[0, :2].tolist() == [0, 1] and cache.table[1, :3].tolist() == [2, 3, 4] and cache.ref.tolist() == [1] * 5 + [0] * 45


def test_fork_refuses_and_runs_out():
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, _ = kv.make_cache(4, [40, 0, 0, 32, 0, 0, 0], [0] * 7, page=16, spare=1, max_pages=5)
    plain = Plain(cache, 16)
    parent = [-1, 0, 0, -1, 3, 2, 9]  # one page for two copies; one that needs none; a copy's copy; a slot that is not there
    done = ab.cache_fork(cache, kv.i32(parent))
    torch.cuda.synchronize()
    assert done.tolist() == [0, 1, 0, 0, 1, 0, 0]
    assert plain.fork(parent[:6] + [-1]) == done.tolist()
    plain.check(cache, 9)
    cache.status.zero_()
    ab.cache_fork(cache, kv.i32([-1, -1, -1, 0, -1, -1, -1]))  # slot 3 holds pages
    plain.check(cache, 9)


def test_compact_refuses():
    """a slot whose path cannot be followed is left as it is, the others go on"""
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, rooms = [30, 20, 10, 5, 40, 3, 8], [20] * 7
    cache, _ = kv.make_cache(5, lens, rooms, page=16, layers=2)
    cache.ref[cache.table[4, 2].long()] += 1  # slot 4's page of places 32 .. 47 has another holder
    plain = Plain(cache, 16)
    kept = np.array([3, 3, 3, 3, 2, 5, 3])
    path = np.array([[0, 2, 5, -1], [0, 5, 5, -1], [1, 0, 2, -1], [0, 2, 60, -1], [0, 3, -1, -1], [0, 1, 2, 3], [0, -1, 3, 4]])
    ab.cache_compact(cache, kv.i32(kept), kv.i32(path))
    state = (plain.used.copy(), plain.table.copy())
    plain.compact([3, 0, 0, 0, 0, 0, 0], path)
    for s in range(1, 7):  # (left as they are: their room is still theirs)
        gone = state[1][s, plain.used[s] : state[0][s]]
        plain.table[s], plain.used[s] = state[1][s], state[0][s]
        np.add.at(plain.ref, gone, 1)
    plain.check(cache, 9)


def test_free_reports_lists_that_do_not_fit():
    import arcinfer_b200 as ab
    import kvutil as kv

    for what in ("page", "holders", "used"):
        cache, _ = kv.make_cache(6, [40, 20], [0, 0], page=16)
        if what == "page":
            cache.table[0, 1] = 10**6
        elif what == "holders":
            cache.ref[cache.table[0, 1].long()] = 0
        else:
            cache.used[0] = 10**6
        ab.cache_free(cache, kv.i32([1, 1]))
        torch.cuda.synchronize()
        assert int(cache.status.item()) == 9 and int(cache.used[1].item()) == 0 and int(cache.ref.min().item()) == 0, what


# ---------------------------------------------------------------- append
def _append64(x, w, pos, inv_freq, rot, interleaved, eps):
    """norm and rotation of [T, H, dim] in 64 bits"""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(dim=2, keepdim=True) + eps).sqrt() * w.double()
    angle = (pos.double()[:, None] * inv_freq)[:, None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    h = rot // 2
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :h], y[..., h:rot])
    r, size = y.clone(), y.abs()
    big = a.abs() + b.abs()
    if interleaved:
        r[..., 0:rot:2], r[..., 1:rot:2] = a * c - b * s, a * s + b * c
        size[..., 0:rot:2] = size[..., 1:rot:2] = big
    else:
        r[..., :h], r[..., h:rot] = a * c - b * s, a * s + b * c
        size[..., :h] = size[..., h:rot] = big
    return r, size


def _near(got, want, size, dtype):
    """half a step of rounding (relative, or among the subnormal numbers); 32-bit work: 2^-19 of the pair (the angle's turn is rounded to 2^-24 of a
    half circle, sine and cosine to 2^-23, the norm's sum, root and products to some 2^-21)"""
    import kvutil as kv

    err = (got.double() - want).abs()
    bound = kv.HALF_STEP[dtype] * want.abs() + 2.0**-19 * size + kv.SMALLEST[dtype]
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,Hq,heads,dtype,layout", [(64, 64, 8, 1, "bf16", "heads"), (64, 16, 5, 5, "fp16", "tokens"), (128, 128, 7, 2, "bf16", "gap"), (128, 96, 32, 8, "fp16", "heads"),
                                                           (128, 0, 4, 2, "bf16", "pages"), (256, 256, 3, 1, "fp16", "heads"), (256, 64, 16, 2, "bf16", "tokens")])
def test_append(dim, rot, Hq, heads, dtype, layout, interleaved):
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [0, 15, 16, 200, 31, 1], [1, 40, 0, 300, 17, 64]
    dt = kv.DTYPES[dtype]
    cache, _ = kv.make_cache(dim + rot, lens, nodes, heads, 16, dim, dt, layers=2, layout=layout)
    cache.k.fill_(3.0), cache.v.fill_(3.0)
    off = np.concatenate([[0], np.cumsum(nodes)])
    T = int(off[-1])
    gen = torch.Generator(device="cuda")
    gen.manual_seed(dim)
    qkv = (torch.randn(T + 2, (Hq + 2 * heads) * dim, generator=gen, device="cuda") * 3).to(dt)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([Hq * dim, heads * dim, heads * dim], dim=1))
    qw, kw = (1 + 0.3 * torch.randn(2, dim, generator=gen, device="cuda")).unbind(0)
    pos = torch.randint(0, 1 << 20, (T + 2,), generator=gen, device="cuda", dtype=torch.int32)
    pos[0], pos[1] = 0, 2**31 - 1
    inv = torch.from_numpy(1e4 ** (-np.arange(0, rot, 2) / max(rot, 1))).cuda()
    before = qkv.clone()
    for weights in ((qw, kw), (None, kw), (None, None)):
        out = torch.full((T + 2, Hq, dim), 9.0, dtype=dt, device="cuda")
        got = ab.cache_append(cache, q, k, v, kv.i32(off), pos, inv, layer=1, q_weight=weights[0], k_weight=weights[1], eps=1e-5, interleaved=interleaved, q_out=out)
        torch.cuda.synchronize()
        assert got is out and int(cache.status.item()) == 0 and torch.equal(qkv, before)
        _near(out[:T], *_append64(q[:T], weights[0], pos[:T], inv, rot, interleaved, 1e-5), dt)
        assert (out[T:] == 9.0).all()
        wk, size = _append64(k[:T], weights[1], pos[:T], inv, rot, interleaved, 1e-5)
        written = torch.zeros(cache.k.shape[1:4], dtype=torch.bool, device="cuda")
        for s, n in enumerate(lens):
            place = n + torch.arange(nodes[s], device="cuda")
            page = cache.table[s].long()[place // 16]
            a, b = int(off[s]), int(off[s + 1])
            _near(cache.k[1][page, :, place % 16], wk[a:b], size[a:b], dt)
            assert torch.equal(cache.v[1][page, :, place % 16], v[a:b])
            written[page, :, place % 16] = True
        assert (cache.k[1][~written] == 3.0).all() and (cache.v[1][~written] == 3.0).all() and (cache.k[0] == 3.0).all() and (cache.v[0] == 3.0).all()
    # in place
    ab.cache_append(cache, q, k, v, kv.i32(off), pos, inv, layer=1, eps=1e-5, interleaved=interleaved, q_out=q)
    torch.cuda.synchronize()
    assert torch.equal(q[:T], out[:T]) and torch.equal(q[T:], before[T:, : Hq * dim].unflatten(1, (-1, dim)))


def test_append_rows_of_zeros_and_extremes():
    """a row of zeros has no direction (eps keeps it at zero); large values whose squares would leave 16 bits"""
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, _ = kv.make_cache(1, [0], [3], 1, 16, 128, torch.float16)
    x = torch.zeros(3, 1, 128, dtype=torch.float16, device="cuda")
    x[1] = 60000.0
    x[2] = 2.0**-20
    w = torch.ones(128, device="cuda")
    inv = torch.from_numpy(1e4 ** (-np.arange(0, 128, 2) / 128)).cuda()
    pos = kv.i32([5, 0, 0])
    out = ab.cache_append(cache, x, x, x, kv.i32([0, 3]), pos, inv, q_weight=w, k_weight=w, eps=1e-6)
    torch.cuda.synchronize()
    assert (out[0] == 0).all() and (out[1] == 1.0).all()
    _near(out, *_append64(x, w, pos, inv, 128, False, 1e-6), x.dtype)


def test_append_reports_places_outside_the_pages():
    import arcinfer_b200 as ab
    import kvutil as kv

    for what in ("room", "page", "length"):
        cache, _ = kv.make_cache(2, [30, 5], [2, 8], 2, 16, 64)
        cache.k.fill_(1.0), cache.v.fill_(1.0)
        if what == "page":
            cache.table[0, 1] = -1
        if what == "length":
            cache.length[0] = -40
        n = 3 if what == "room" else 2  # (places 30, 31 lie in the slot's pages, 32 does not)
        x = torch.full((n + 8, 2, 64), 2.0, dtype=torch.bfloat16, device="cuda")
        ab.cache_append(cache, x, x, x, kv.i32([0, n, n + 8]), kv.i32(np.zeros(n + 8)), torch.zeros(0, dtype=torch.float64, device="cuda"))
        torch.cuda.synchronize()
        assert int(cache.status.item()) == 9, what
        assert int((cache.v == 2.0).sum().item()) == (8 + (2 if what == "room" else 0)) * 2 * 64, what
