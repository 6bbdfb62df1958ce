"""The walk over a tree of drafts against a plain one; and a whole step of a server over the paged cache."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _walk(token, draft, parent):
    path = [0]
    while True:
        here = path[-1]
        child = [i for i in range(1, len(token)) if parent[i] == here and i > here and draft[i] == token[here]]
        if not child:
            return path, token[here]
        path.append(child[0])


@pytest.mark.parametrize("slots,most", [(1, 1), (1, 8), (7, 33), (513, 64)])
def test_against_a_plain_walk(slots, most):
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(slots + most)
    for vocab in (1, 2, 5):
        n = g.integers(0 if slots > 1 else 1, most + 1, slots)
        n[-1] = most
        off = np.concatenate([[0], np.cumsum(n)])
        T = int(off[-1])
        token, draft = g.integers(0, vocab, T), g.integers(0, vocab, T)
        at = np.arange(T) - np.repeat(off[:-1], n)
        parent = np.where(at == 0, -1, np.maximum(0, at - 1 - g.integers(0, 4, T)))
        odd = g.random(T) < 0.05  # nodes that hang on nothing, or on a later node: never reached
        parent = np.where(odd & (at > 0), g.choice([-1, 63, -5], T), parent)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = {k: v.cpu().numpy() for k, v in ab.accept_tree(kv.i32(token), kv.i32(draft), kv.i32(parent), kv.i32(off), most, status=status).items()}
        assert int(status.item()) == 0
        for s in range(slots):
            a, b = off[s], off[s + 1]
            path, nxt = _walk(token[a:b], draft[a:b], parent[a:b]) if b > a else ([], -1)
            assert (got["accepted"][s], got["kept"][s], got["next"][s]) == (len(path) - 1, len(path), nxt), s
            assert got["path"][s].tolist() == path + [-1] * (most - len(path)), s


def test_a_chain_is_accept_batch():
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(3)
    n = g.integers(1, 9, 20)
    off = np.concatenate([[0], np.cumsum(n)])
    token, draft = g.integers(0, 2, off[-1]), g.integers(0, 2, off[-1])
    parent = np.arange(off[-1]) - np.repeat(off[:-1], n) - 1
    got = ab.accept_tree(kv.i32(token), kv.i32(draft), kv.i32(parent), kv.i32(off), 8)
    drafts = np.concatenate([draft[off[s] + 1 : off[s + 1]] for s in range(20)])
    acc, nxt = ab.accept_batch(kv.i32(token), kv.i32(off), kv.i32(drafts), kv.i32(off - np.arange(21)))
    assert torch.equal(got["accepted"], acc) and torch.equal(got["next"], nxt)


def test_lists_that_do_not_fit_are_reported():
    import arcinfer_b200 as ab
    import kvutil as kv

    z = kv.i32(np.zeros(10))
    for off, most in (([0, 5, 11], 8), ([0, 5, 10], 4), ([0, 7, 3], 8)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = ab.accept_tree(z, z, z, kv.i32(off), most, status=status)
        assert int(status.item()) == 9 and got["kept"][1].item() == 0 and got["next"][1].item() == -1


def _model(seed, layers, Hq, heads, dim, V, width):
    """a small stack of attention layers and a head, as a server would run them with the library's calls around"""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=gen, device="cuda")  # noqa: E731
    return dict(embed=r(V, width), qkv=[r(width, (Hq + 2 * heads) * dim) / width**0.5 for _ in range(layers)], out=[r(Hq * dim, width) / (Hq * dim) ** 0.5 for _ in range(layers)],
                head=r(width, V) * 0.3, w=[1 + 0.1 * r(2, dim) for _ in range(layers)], inv=torch.from_numpy(1e4 ** (-np.arange(0, dim, 2) / dim)).cuda(), Hq=Hq, heads=heads, dim=dim,
                layers=layers)


def _forward(m, cache, tokens, off, depth, mask, most):
    import arcinfer_b200 as ab

    x = m["embed"][tokens.long()]
    slot = torch.repeat_interleave(torch.arange(cache.slots, device="cuda"), (off[1:] - off[:-1]).long())
    pos = (cache.length[slot] + depth).int()
    Hq, heads, dim = m["Hq"], m["heads"], m["dim"]
    for layer in range(m["layers"]):
        qkv = (x @ m["qkv"][layer]).to(cache.dtype)
        q, k, v = (y.unflatten(1, (-1, dim)) for y in qkv.split([Hq * dim, heads * dim, heads * dim], dim=1))
        q = ab.cache_append(cache, q, k, v, off, pos, m["inv"], layer=layer, q_weight=m["w"][layer][0].contiguous(), k_weight=m["w"][layer][1].contiguous())
        a = ab.tree_attention(q, cache, off, most, mask=mask, layer=layer)["out"]
        x = x + a.flatten(1).float() @ m["out"][layer]
    return (x @ m["head"]).contiguous()


@pytest.mark.parametrize("dim,dtype", [(64, "fp16"), (128, "bf16"), (256, "fp16")])
def test_a_whole_step(dim, dtype):
    """Prompts token by token (single nodes) against the same tokens given as a tree: reserve, append,
    attention, argmax, acceptance, compaction; then the next step over the compacted cache, and a copy of
    a slot, see the same texts."""
    import arcinfer_b200 as ab
    import kvutil as kv

    dt, V, S = kv.DTYPES[dtype], 500, 3
    m = _model(dim, 2, 4, 2, dim, V, 96)
    g = np.random.default_rng(dim)
    tree = ab.kvcache.KVCache.empty(2, 60, 2, 16, dim, S + 1, 8, dt)
    line = ab.kvcache.KVCache.empty(2, 60, 2, 16, dim, S + 1, 8, dt)

    def single(cache, tokens):
        """one token of every slot (-1: none)"""
        live = [int(t >= 0) for t in tokens]
        off = kv.i32(np.concatenate([[0], np.cumsum(live)]))
        ab.cache_reserve(cache, kv.i32(live))
        lg = _forward(m, cache, kv.i32([t for t in tokens if t >= 0]), off, torch.zeros(sum(live), dtype=torch.int32, device="cuda"), None, 1)
        ab.cache_compact(cache, kv.i32(live), kv.i32(np.zeros((S + 1, 1))))
        return lg

    texts = [list(g.integers(0, V, n)) for n in (13, 15, 20)]
    for i in range(20):
        now = [t[i] if i < len(t) else -1 for t in texts] + [-1]
        single(tree, now), single(line, now)
    assert tree.length.tolist() == [13, 15, 20, 0]
    # the line's continuation: what greedy decoding gives after a certain root
    roots = [int(x) for x in g.integers(0, V, S)]
    want, now = [[] for _ in range(S)], list(roots)
    for _ in range(5):
        lg = single(line, now + [-1])
        now = [int(t) for t in ab.argmax_batch(lg)["argmax"]]
        for s in range(S):
            want[s].append(now[s])
    # trees: the right drafts down to some depth, on wrong branches' later siblings, between wrong ones
    parents, drafts, good = [], [], [2, 4, 0]
    for s in range(S):
        par, dr, at = [-1], [roots[s]], 0
        for d in range(good[s]):
            for wrong in range(2):
                par.append(at), dr.append((want[s][d] + 1 + wrong) % V)
            par.append(at), dr.append(want[s][d])
            at = len(par) - 1
        par.append(at), dr.append((want[s][good[s]] + 7) % V)
        parents.append(par), drafts.append(dr)
    off, parent, depth, mask = ab.tree_lists(parents + [[]])
    n = np.diff(off)
    ab.cache_reserve(tree, kv.i32(n))
    dr = kv.i32(np.concatenate(drafts))
    lg = _forward(m, tree, dr, kv.i32(off), kv.i32(depth), torch.from_numpy(mask).cuda(), 64)
    tok = ab.argmax_batch(lg)["argmax"]
    acc = ab.accept_tree(tok, dr, kv.i32(parent), kv.i32(off), 64)
    assert acc["accepted"].tolist() == good + [-1]
    assert acc["next"].tolist()[:S] == [want[s][good[s]] for s in range(S)]
    ab.cache_compact(tree, acc["kept"], acc["path"])
    torch.cuda.synchronize()
    assert tree.length.tolist() == [13 + 3, 15 + 5, 20 + 1, 0] and int(tree.status.item()) == 0 and int(line.status.item()) == 0
    assert int((tree.ref > 0).sum().item()) == 1 + 2 + 2
    # the compacted keys and values are the line's
    for s in range(S):
        place = torch.arange(int(tree.length[s].item()), device="cuda")
        for a, b in ((tree.k, line.k), (tree.v, line.v)):
            x, y = (c[:, t[s].long()[place // 16], :, place % 16].float() for c, t in ((a, tree.table), (b, line.table)))
            assert (x - y).norm() <= 0.02 * y.norm(), s  # (two layers of results rounded to 16 bits along different sums)
    # a copy goes on as its parent does
    ab.cache_fork(tree, kv.i32([-1, -1, -1, 1]))
    nxt = acc["next"].tolist()
    lg = single(tree, nxt[:S] + [nxt[1]])
    assert torch.equal(lg[1], lg[3]) and int(tree.status.item()) == 0
    ab.cache_free(tree, kv.i32([1] * (S + 1)))
    torch.cuda.synchronize()
    assert int(tree.ref.sum().item()) == 0


def test_a_step_captured_and_replayed():
    """reserve, append, attention, acceptance and compaction in one graph, replayed over a growing cache on a stream
    of its own, against the same calls one by one"""
    import arcinfer_b200 as ab
    import kvutil as kv

    S, N, heads, Hq, dim, layers = 5, 9, 2, 8, 128, 3
    g = np.random.default_rng(9)
    lens = [0, 17, 200, 16, 63]
    off, parent, depth, mask = ab.tree_lists([kv.random_parents(g, N) for _ in range(S)])
    T = int(off[-1])
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    qkv = torch.randn(layers, T, Hq + 2 * heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
    token, draft = kv.i32(g.integers(0, 2, T)), kv.i32(g.integers(0, 2, T))
    slot = torch.from_numpy(np.repeat(np.arange(S), N)).cuda()
    off, parent, depth, mask = kv.i32(off), kv.i32(parent), kv.i32(depth), torch.from_numpy(mask).cuda()
    inv = torch.from_numpy(1e4 ** (-np.arange(0, dim, 2) / dim)).cuda()
    room = kv.i32([N] * S)

    def step(cache):
        ab.cache_reserve(cache, room)
        pos = cache.length[slot] + depth
        outs = []
        for layer in range(layers):
            q, k, v = qkv[layer].split([Hq, heads, heads], dim=1)
            q = ab.cache_append(cache, q, k, v, off, pos, inv, layer=layer)
            outs.append(ab.tree_attention(q, cache, off, N, mask=mask, layer=layer)["out"])
        acc = ab.accept_tree(token, draft, parent, off, N)
        ab.cache_compact(cache, acc["kept"], acc["path"])
        return outs, acc

    a, b = (kv.make_cache(3, lens, [0] * S, heads, 16, dim, layers=layers, spare=40, max_pages=24)[0] for _ in range(2))
    fresh = [x.clone() for x in (b.k, b.v, b.table, b.used, b.ref, b.length)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b)  # (before the capture, once)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs, acc = step(b)
    torch.cuda.synchronize()
    for x, y in zip((b.k, b.v, b.table, b.used, b.ref, b.length), fresh):
        x.copy_(y)
    for _ in range(4):
        want, wacc = step(a)
        graph.replay()
        torch.cuda.synchronize()
        assert int(a.status.item()) == 0 and int(b.status.item()) == 0
        for x, y in zip(outs + list(acc.values()), want + list(wacc.values())):
            assert torch.equal(x, y)
        for name in ("table", "used", "ref", "length"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
        for x, y in ((a.k, b.k), (a.v, b.v)):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    assert a.length.tolist() != lens
