"""Tree attention over a paged cache against sums in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [0, 1, 15, 63, 64, 65, 127, 128, 129, 700, 0, 1001]


def _case(seed, lens, nodes, Hq, heads=2, page=16, dim=128, dtype=torch.bfloat16, layout="heads", layers=1, chain=False, back=4):
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(seed)
    cache, rows = kv.make_cache(seed, lens, nodes, heads, page, dim, dtype, layers, layout)
    off, parent, depth, mask = ab.tree_lists([kv.random_parents(g, n, 1 if chain else back) for n in nodes])
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)
    q = (torch.randn(int(off[-1]), Hq, dim, generator=gen, device="cuda") * 1.5).to(dtype)
    return cache, rows, off, [int(m) & (2**64 - 1) for m in mask], torch.from_numpy(mask).cuda(), q


def _check(cache, rows, off, masks, q, got, lens, scale=None, layer=0):
    import kvutil as kv

    assert int(cache.status.item()) == 0
    kv.check_attention(got["out"], got.get("lse"), q, rows, lens, off, masks, cache.dim**-0.5 if scale is None else scale, layer)


@pytest.mark.parametrize("layout", ["heads", "tokens", "gap", "odd"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,page,Hq,heads", [(64, 16, 8, 8), (64, 256, 8, 1), (128, 16, 14, 2), (128, 32, 2, 2), (128, 64, 32, 2), (128, 128, 10, 2), (256, 16, 4, 4), (256, 64, 16, 2)])
def test_against_64_bits(dim, page, Hq, heads, dtype, layout):
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(dim + page + Hq)
    nodes = [int(x) for x in g.integers(1, 17, len(LENS))]
    cache, rows, off, masks, mask, q = _case(dim + page, LENS, nodes, Hq, heads, page, dim, kv.DTYPES[dtype], layout)
    got = ab.tree_attention(q, cache, kv.i32(off), 16, mask=mask, want_lse=True)
    _check(cache, rows, off, masks, q, got, LENS)


@pytest.mark.parametrize("dim,Hq,heads", [(64, 16, 2), (128, 16, 2), (128, 10, 2), (256, 6, 2), (128, 64, 1)])
def test_large_trees(dim, Hq, heads):
    """64 nodes a slot (the last bit of a mask in use), several tiles of rows"""
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [0, 300, 64, 1000], [64, 64, 63, 33]
    cache, rows, off, masks, mask, q = _case(dim + Hq, lens, nodes, Hq, heads, 32, dim, back=9)
    got = ab.tree_attention(q, cache, kv.i32(off), 64, mask=mask, want_lse=True)
    _check(cache, rows, off, masks, q, got, lens)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,Hq,heads,most", [(64, 16, 8, 6), (64, 40, 8, 40), (128, 16, 8, 6), (128, 40, 8, 40), (256, 16, 8, 6), (256, 40, 8, 30)])
def test_many_short_texts(dim, Hq, heads, most, dtype):
    """several items, whole and cut, of one tile and of several, for every CTA"""
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(dim + Hq)
    slots = 40
    lens = [int(x) for x in g.choice([0, 3, 100, 120, 129, 250, 300, 380, 500, 640, 900], slots)]
    nodes = [int(x) for x in g.integers(0, most + 1, slots)]
    cache, rows, off, masks, mask, q = _case(dim + Hq, lens, nodes, Hq, heads, 32, dim, kv.DTYPES[dtype])
    for _ in range(3):
        got = ab.tree_attention(q, cache, kv.i32(off), most, mask=mask, want_lse=True)
        _check(cache, rows, off, masks, q, got, lens)
    same = q.clone()  # results in place of the queries
    assert torch.equal(ab.tree_attention(same, cache, kv.i32(off), most, mask=mask, out=same)["out"], got["out"])


@pytest.mark.parametrize("slots", [129, 700])
def test_many_slots(slots):
    """more slots than a warp adds up on its own"""
    import arcinfer_b200 as ab
    import kvutil as kv

    for dim, Hq in ((64, 8), (128, 2), (128, 48), (256, 4)):
        g = np.random.default_rng(slots + dim)
        lens = [int(x) for x in g.integers(0, 200, slots)]
        lens[slots // 2] = 5000
        nodes = [int(x) for x in g.choice([0, 0, 1, 2, 7], slots)]
        cache, rows, off, masks, mask, q = _case(dim, lens, nodes, Hq, 2, 16, dim)
        got = ab.tree_attention(q, cache, kv.i32(off), 7, mask=mask, want_lse=True)
        _check(cache, rows, off, masks, q, got, lens)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length", [1, 40, 128, 129, 5000, 40000])
def test_single_tokens(dim, length):
    """one slot, one new token: the texts are cut over the whole machine and joined"""
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, rows, off, masks, _, q = _case(length, [length], [1], 8, 2, 64, dim)
    got = ab.tree_attention(q, cache, kv.i32(off), 1, want_lse=True)
    _check(cache, rows, off, masks, q, got, [length])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chains_scales_and_layers(dim):
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [77, 0, 513], [64, 40, 9]
    cache, rows, off, masks, _, q = _case(5, lens, nodes, 4, 2, 16, dim, layers=3, layout="pages", chain=True)
    for layer in (0, 2):
        got = ab.tree_attention(q, cache, kv.i32(off), 64, layer=layer, scale=0.031, want_lse=True)
        _check(cache, rows, off, masks, q, got, lens, 0.031, layer)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_see_nothing_and_rows_that_skip_themselves(dim):
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [0, 0, 200], [5, 64, 12]
    cache, rows, off, masks, _, q = _case(6, lens, nodes, 8, 2, 16, dim)
    g = np.random.default_rng(6)
    masks = [int(x) for x in g.integers(0, 2**63, len(masks))]  # any nodes, itself or not, some that are not there
    for t in (0, 3, 7, 30, 70):
        masks[t] = 0
    masks[4] = 1 << 40  # a node that the slot does not have
    masks[5] = 2**64 - 1
    got = ab.tree_attention(q, cache, kv.i32(off), 64, mask=torch.from_numpy(np.asarray(masks, np.uint64).view(np.int64)).cuda(), want_lse=True)
    _check(cache, rows, off, masks, q, got, lens)
    for t in (0, 3, 4, 7, 30):  # (row 70 still has its 200 tokens)
        assert (got["out"][t] == 0).all() and (got["lse"][t] == -float("inf")).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,bad", [(64, "nan"), (128, "nan"), (128, "inf"), (256, "-inf")])
def test_masked_nodes_have_no_influence(dim, bad, dtype):
    """NaN and infinities in nodes that only some rows see: those rows show them where they stand, the others are as ever"""
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [100, 0, 130, 3], [20, 9, 64, 7]
    cache, rows, off, masks, mask, q = _case(7, lens, nodes, 8, 2, 16, dim, kv.DTYPES[dtype])
    hit = [3, 8, 63, 6]
    for s, j in enumerate(hit):
        place = lens[s] + j
        page = int(cache.table[s, place // 16].item())
        cache.v[0, page, :, place % 16, 5:9] = float(bad)
        if bad == "nan":
            cache.k[0, page, :, place % 16, 1] = float(bad)
    clean = [[k.clone(), v.clone()] for k, v in rows]
    got = ab.tree_attention(q, cache, kv.i32(off), 64, mask=mask, want_lse=True)
    torch.cuda.synchronize()
    sees = torch.tensor([bool((masks[t] >> hit[s]) & 1) for s in range(4) for t in range(off[s], off[s + 1])], device="cuda")
    assert sees.any() and not sees.all()
    touched = got["out"][sees]
    if bad == "nan":
        assert torch.isnan(touched).all() and torch.isnan(got["lse"][sees]).all()
    else:
        assert (touched[:, :, 5:9] == float(bad)).all()
        assert torch.isfinite(touched[:, :, :5]).all() and torch.isfinite(touched[:, :, 9:]).all()
        # the other values of such rows are as without it
        fine = got["out"].clone()
        fine[:, :, 5:9] = 0
        for k, v in clean:
            v[..., 5:9] = 0
        kv.check_attention(fine, got["lse"], q, clean, lens, off, masks, dim**-0.5)
        return
    # rows that do not see it, with it out of the comparison for those that do
    got["out"][sees], masks = 0, [0 if sees[t] else m for t, m in enumerate(masks)]
    for s in range(4):
        a, b = int(off[s]), int(off[s + 1])
        want, wl, size = kv.attention64(q[a:b], rows[s][0][0], rows[s][1][0], lens[s], masks[a:b], dim**-0.5)
        free = ~sees[a:b]
        err = (got["out"][a:b].double() - want).abs()[free]
        u = kv.HALF_STEP[q.dtype]
        assert (err <= u * want.abs()[free] + (u + 2.0**-16) * size[free] + 100 * kv.SMALLEST[q.dtype]).all(), s


def test_large_and_small_scores():
    """scores that rise by hundreds along the text, and ones that all but one place loses to"""
    import arcinfer_b200 as ab
    import kvutil as kv

    for dim, dtype in ((64, "fp16"), (128, "bf16"), (256, "fp16")):
        cache, rows, off, masks, mask, q = _case(8, [900, 2000], [8, 3], 8, 2, 16, dim, kv.DTYPES[dtype])
        # the keys grow along the text, so that the running maximum keeps rising; 2^7 a score at most
        for s, n in enumerate((900, 2000)):
            k = rows[s][0]
            k *= torch.linspace(0.01, 2.0, k.shape[2], device="cuda")[None, None, :, None].to(k.dtype)
            place = torch.arange(k.shape[2], device="cuda")
            pages = cache.table[s].long()[place // 16]
            cache.k[0][pages, :, place % 16] = k[0].transpose(0, 1)
        got = ab.tree_attention(q, cache, kv.i32(off), 8, mask=mask, want_lse=True, scale=0.2)
        _check(cache, rows, off, masks, q, got, [900, 2000], 0.2)


def test_strides_slots_without_work_and_rows_behind_the_last():
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [33, 50, 0, 200, 5], [4, 0, 3, 0, 6]
    cache, rows, off, masks, mask, q = _case(9, lens, nodes, 6, 2, 16, 128)
    T = int(off[-1])
    wide = torch.zeros(T + 3, 6 * 128 + 40, dtype=q.dtype, device="cuda")  # queries inside wider rows
    wide[:T, : 6 * 128] = q.reshape(T, -1)
    first = torch.full((6, T + 3, 136), 7.0, dtype=q.dtype, device="cuda")  # results head by head, with gaps
    out = first.transpose(0, 1)[:, :, :128]
    got = ab.tree_attention(wide[:, : 6 * 128].unflatten(1, (6, 128)), cache, kv.i32(off), 8, mask=torch.cat([mask, mask[:3]]), out=out)
    assert got["out"] is out
    _check(cache, rows, off, masks, q, {"out": out[:T]}, lens)
    assert (out[T:] == 7.0).all() and (first[:, :, 128:] == 7.0).all()


def test_pool_beyond_32_bits():
    """pages whose byte offsets pass 2^32"""
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, rows, off, masks, mask, q = _case(10, [600], [5], 8, 2, 256, 256)
    n = 9000  # pages of 2 heads x 256 rows x 512 bytes: 2.36e9 values a pool
    far = [torch.empty(1, n, 2, 256, 256, dtype=q.dtype, device="cuda") for _ in range(2)]
    table = cache.table.clone()
    used = int(cache.used[0].item())
    for i in range(used):
        p = int(table[0, i].item())
        for x, y in zip(far, (cache.k, cache.v)):
            x[0, n - 1 - i] = y[0, p]
        table[0, i] = n - 1 - i
    big = ab.KVCache(*far, table, cache.used, kv.i32(np.zeros(n)), cache.length)
    got = ab.tree_attention(q, big, kv.i32(off), 8, mask=mask, want_lse=True)
    _check(big, rows, off, masks, q, got, [600])


def test_streams_and_graphs():
    """two captured calls and an eager one at the same time, each with its own scratch; replays give what the first call gave"""
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [9000, 20], [6, 12]
    cases = [_case(20 + i, lens, nodes, 8, 2, 16, 128) for i in range(3)]
    offs = [kv.i32(c[2]) for c in cases]
    call = lambda i: ab.tree_attention(cases[i][5], cases[i][0], offs[i], 12, mask=cases[i][4], want_lse=True)  # noqa: E731
    first = [{k: v.clone() for k, v in call(i).items()} for i in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i < 2:
                    graphs[i].replay()
                else:
                    last = call(2)
    torch.cuda.synchronize()
    for i, got in enumerate(outs + [last]):
        for k in ("out", "lse"):
            assert torch.equal(got[k], first[i][k]), (i, k)
        _check(cases[i][0], cases[i][1], cases[i][2], cases[i][3], cases[i][5], got, lens)


def test_same_results_every_time():
    import arcinfer_b200 as ab
    import kvutil as kv

    cache, rows, off, masks, mask, q = _case(30, [3000, 17, 800], [9, 16, 2], 16, 2, 32, 128)
    a = ab.tree_attention(q, cache, kv.i32(off), 16, mask=mask, want_lse=True)
    for _ in range(10):
        b = ab.tree_attention(q, cache, kv.i32(off), 16, mask=mask, want_lse=True)
        assert torch.equal(a["out"], b["out"]) and torch.equal(a["lse"], b["lse"])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_lists_that_do_not_fit_are_reported(dim):
    """a page that is not there, a slot with fewer pages than its tokens, more nodes than were announced: a status, no access"""
    import arcinfer_b200 as ab
    import kvutil as kv

    lens, nodes = [100, 40], [4, 4]
    for what in ("page", "page below", "used", "length", "nodes", "rows"):
        cache, rows, off, masks, mask, q = _case(40, lens, nodes, 4, 2, 16, dim)
        limit = 4
        if what == "page":
            cache.table[1, 1] = cache.k.shape[1]
        elif what == "page below":
            cache.table[1, 0] = -1
        elif what == "used":
            cache.used[1] = 2
        elif what == "length":
            cache.length[1] = -3
        elif what == "nodes":
            limit = 3
        else:
            off = off.copy()
            off[2] = 9  # (q has eight rows)
        ab.tree_attention(q, cache, kv.i32(off), limit, mask=mask)
        torch.cuda.synchronize()
        assert int(cache.status.item()) == 9, what
