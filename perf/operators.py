"""The operators around the verification of drafted tokens over a paged cache: the cache's pages
(reserve, compact, fork, free), the norm and rotation that write queries and keys, the attention of
a tree of drafts, and the walk that accepts a path of it.

A case is a dict of plain values; `kind` names the operator:
  attention  tree_attention: every slot's drafted nodes attend to its cached tokens and to their ancestors
  append     cache_append: norm of queries and keys for each head, rotation by position, keys and values to their pages
  step       cache_reserve + cache_compact: room for the drafted nodes, the kept ones moved together, pages given back
  fork       cache_free + cache_fork: the copies of some slots are dropped and made again
  accept     accept_tree: the path of drafts that agree with the tokens chosen

With `own` false, `run` computes these in elementary torch operations, in 32 bits (angles in 64).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one request, one new token: the smallest step there is
        dict(name="attention-token", kind="attention", slots=1, nodes=1, ctx=4096, spread=0.0, Hq=32, Hkv=8, D=128, page=16, type="bf16"),
        # one request far into a long text, a tree of 24 drafts, few wide key heads
        dict(name="attention-long", kind="attention", slots=1, nodes=24, ctx=131071, spread=0.0, Hq=16, Hkv=2, D=256, page=64, type="bf16"),
        # a server's batch: ragged texts and trees, seven query heads to a key head
        dict(name="attention-batch", kind="attention", slots=48, nodes=12, ctx=9001, spread=0.95, Hq=28, Hkv=4, D=128, page=32, type="fp16"),
        # the widest verification: 64 nodes a slot, eight query heads to a key head
        dict(name="attention-wide", kind="attention", slots=32, nodes=64, ctx=8192, spread=0.5, Hq=64, Hkv=8, D=128, page=128, type="bf16"),
        # the drafted nodes of a server's batch on their way into the cache
        dict(name="append-step", kind="append", slots=32, nodes=16, ctx=700, spread=0.9, Hq=32, Hkv=8, D=128, page=16, type="bf16", rot=128, pairs="halves", norm=True),
        # whole prompts, a part of each head rotated, positions far into a text
        dict(name="append-prompts", kind="append", slots=8, nodes=2100, ctx=500000, spread=0.3, Hq=16, Hkv=2, D=256, page=64, type="fp16", rot=64, pairs="neighbours", norm=True),
        # what follows one request's verification, over all layers of a model
        dict(name="step-one", kind="step", slots=1, nodes=24, kept=5, ctx=1000, spread=0.0, layers=32, Hkv=4, D=128, page=16, type="bf16"),
        # the same for a server's batch
        dict(name="step-many", kind="step", slots=64, nodes=40, kept=8, ctx=257, spread=0.8, layers=32, Hkv=8, D=128, page=16, type="bf16"),
        # a request that goes on in two ways
        dict(name="fork-one", kind="fork", parents=1, children=1, ctx=1000, rest=9, layers=32, Hkv=4, D=128, page=16, type="fp16"),
        # several answers to each of several requests
        dict(name="fork-many", kind="fork", parents=16, children=3, ctx=400, rest=50, layers=32, Hkv=8, D=128, page=64, type="bf16"),
        # the walk for one request, and for a wide batch of large trees
        dict(name="accept-one", kind="accept", slots=1, nodes=8),
        dict(name="accept-many", kind="accept", slots=512, nodes=64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: sizes over the logarithm of their ranges, head layouts, pages and types of all
    kinds, no dearer than the listed ones."""
    kind = rng.choice(["attention", "attention", "attention", "attention", "append", "append", "step", "fork", "accept"])
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, type=rng.choice(["bf16", "fp16"]), page=rng.choice([16, 32, 64, 128, 256]), D=D, Hkv=Hkv)
    if kind == "attention":
        slots = _log_int(rng, 1, 64)
        group = rng.choice([1, 2, 4, 5, 7, 8])
        nodes = _log_int(rng, 1, 64)
        most = min(131071, 32 * 6144 * 8 * 128 // (slots * Hkv * D), 32 * 6144 * 64 * 64 * 128 // (slots * Hkv * group * nodes * D))
        c.update(slots=slots, nodes=nodes, ctx=_log_int(rng, 100, most), spread=0.0 if slots == 1 else round(rng.uniform(0.0, 1.0), 2), Hq=Hkv * group)
    elif kind == "append":
        prompt = rng.random() < 0.5
        slots = _log_int(rng, 1, 16 if prompt else 64)
        heads = Hkv * rng.choice([1, 4, 7, 8])
        nodes = _log_int(rng, 100, min(4096, 16800 * 20 * 256 // (slots * D * (heads + 2 * Hkv)))) if prompt else _log_int(rng, 1, 64)
        c.update(slots=slots, nodes=nodes, ctx=_log_int(rng, 100, 1000000), spread=round(rng.uniform(0.0, 1.0), 2), Hq=heads, rot=rng.choice([D, D, D // 2, D // 4]),
                 pairs=rng.choice(["halves", "neighbours"]), norm=rng.random() < 0.8)
    elif kind == "step":
        nodes = _log_int(rng, 4, 64)
        c.update(slots=_log_int(rng, 1, 64), nodes=nodes, kept=rng.randint(1, max(1, min(8, nodes - 2))), ctx=_log_int(rng, 20, 257), spread=round(rng.uniform(0.0, 0.9), 2),
                 layers=rng.choice([8, 16, 24, 32]), page=rng.choice([16, 32, 64]), D=rng.choice([64, 128]))
    elif kind == "fork":
        page = c["page"]
        c.update(parents=_log_int(rng, 1, 16), children=rng.randint(1, 3), ctx=_log_int(rng, 20, 400) // page * page, rest=rng.randint(1, min(63, page - 1)), layers=rng.choice([8, 16, 24, 32]),
                 D=rng.choice([64, 128]))
    else:
        c = dict(kind=kind, slots=_log_int(rng, 1, 512), nodes=rng.randint(2, 64))
    return c


# ---------------------------------------------------------------- sizes that follow from a case
def _spread(n, most, share, least):
    """n whole numbers from (1 - share) * most to most, evenly spread, the first the largest"""
    part = (np.arange(n) * 0.6180339887498949) % 1.0
    return np.maximum(least, np.floor(most * (1.0 - share * part))).astype(np.int64)


def _lengths(c):
    return _spread(c["slots"], c["ctx"], c["spread"], 1)


def _nodes(c):
    return _spread(c["slots"], c["nodes"], 0.0 if c["kind"] == "step" or c["spread"] == 0.0 else 0.5, 1)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    kind = c["kind"]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    g = np.random.default_rng(seed)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)  # noqa: E731
    if kind == "accept":
        S, N = c["slots"], c["nodes"]
        n = _spread(S, N, 0.5 if S > 1 else 0.0, 1)
        off = np.concatenate([[0], np.cumsum(n)])
        at = np.arange(off[-1]) - np.repeat(off[:-1], n)
        parent = np.where(at == 0, -1, np.maximum(0, at - 1 - g.integers(0, 4, len(at))))
        # half of the drafts are what was chosen at their parents
        token = g.integers(0, 150000, len(at))
        draft = np.where(g.random(len(at)) < 0.5, token[np.repeat(off[:-1], n) + np.maximum(0, parent)], g.integers(0, 150000, len(at)))
        return dict(c=c, token=i32(token), draft=i32(draft), parent=i32(parent), off=i32(off), n=n)

    if kind == "fork":
        P, K, ps = c["parents"], c["children"], c["page"]
        S = P * (1 + K)
        ctx = c["ctx"] // ps * ps + c["rest"]
        length = np.full(S, ctx)
        full = ctx // ps
        own_pages = np.where(np.arange(S) < P, full + 1, 1)  # a copy shares its full pages and has its last one to itself
        used = np.full(S, full + 1)
        layers = c["layers"]
    else:
        S, ps = c["slots"], c["page"]
        length = _lengths(c)
        n = _nodes(c)
        off = np.concatenate([[0], np.cumsum(n)])
        room = n if kind in ("attention", "append") else 0
        # (appended texts begin late in their positions but early in their pages, so that the pool stays small)
        length = length % 1000 if kind == "append" else length
        used = own_pages = -(-(length + room) // ps)
        layers = c.get("layers", 1)
    total = int(own_pages.sum())
    spare = total // 8 + 8 + (S * (c["nodes"] // ps + 2) if kind == "step" else 0)
    order = g.permutation(total + spare)
    first = np.concatenate([[0], np.cumsum(own_pages)])
    table = np.full((S, int(used.max()) + (c["nodes"] // ps + 2 if kind == "step" else 1)), -1)
    for s in range(S):
        table[s, used[s] - own_pages[s] : used[s]] = order[first[s] : first[s + 1]]
    if kind == "fork":
        parent = np.where(np.arange(S) < P, -1, np.arange(S) % P)
        table[P:, :full] = table[parent[P:], :full]
    ref = np.zeros(total + spare, np.int64)
    np.add.at(ref, table[table >= 0], 1)
    shape = (layers, total + spare, c["Hkv"], ps, c["D"])
    dtype = TYPES[c["type"]]
    k, v = (torch.empty(shape, dtype=dtype, device=DEV) for _ in range(2))
    for x in (k, v):
        for layer in range(layers):
            x[layer] = torch.randn(shape[1:], generator=gen, device=DEV)
    s = dict(c=c, k=k, v=v, table=i32(table), used=i32(used), ref=i32(ref), length=i32(length))
    if own:
        import arcinfer_b200 as ab

        s["cache"] = ab.KVCache(k, v, s["table"], s["used"], s["ref"], s["length"])
    if kind == "fork":
        s.update(parent=i32(parent), which=i32(parent >= 0))
        return s
    s.update(off=i32(off), n=n, length_now=length)
    if kind == "step":
        # the kept nodes of every slot: the root and some later ones (its first child was refused, so all of these move)
        K = min(c["kept"], c["nodes"])
        path = np.full((S, c["nodes"]), -1)
        for r in range(S):
            path[r, :K] = np.concatenate([[0], np.sort(g.permutation(np.arange(2, c["nodes"]))[: K - 1])])
        s.update(extra=i32(n), kept=i32(np.full(S, K)), path=i32(path), length_out=torch.zeros(S, dtype=torch.int32, device=DEV))
        return s
    T, Hq, Hkv, D = int(off[-1]), c["Hq"], c["Hkv"], c["D"]
    slot = np.repeat(np.arange(S), n)
    at = np.arange(T) - off[slot]
    if kind == "append":
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=DEV).to(dtype)
        s["q_in"], s["k_in"], s["v_in"] = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        s["q_weight"], s["k_weight"] = (1.0 + 0.2 * torch.randn(2, D, generator=gen, device=DEV)).unbind(0) if c["norm"] else (None, None)
        s["pos"] = i32(_lengths(c)[slot] + at)
        s["inv_freq"] = torch.from_numpy(10000.0 ** (-np.arange(0, c["rot"], 2) / c["rot"])).to(DEV)
        s["slot"], s["at"] = torch.from_numpy(slot).to(DEV), torch.from_numpy(at).to(DEV)
        return s
    # a tree: each node hangs on one of the few before it; a node attends to itself and its ancestors
    up = np.maximum(0, at - 1 - g.integers(0, 4, T))
    sees = np.zeros(T, np.uint64)
    for i in range(c["nodes"]):
        rows = np.flatnonzero(at == i)
        sees[rows] = np.uint64(1 << i) | (sees[rows - i + up[rows]] if i else np.uint64(0))
    # queries about as long as those of trained heads: the scores spread over a few units
    s["q"] = (1.5 * torch.randn(T, Hq, D, generator=gen, device=DEV)).to(dtype)
    s["mask"] = torch.from_numpy(sees.view(np.int64)).to(DEV)
    s["slot"], s["at"] = torch.from_numpy(slot).to(DEV), torch.from_numpy(at).to(DEV)
    return s


# ---------------------------------------------------------------- the plain forms
def _attention(s):
    """softmax(q k / sqrt(D)) v over the cached tokens and the nodes that a node's mask names, in 32
    bits: the pages of all slots gathered side by side, scores of masked places -inf."""
    c = s["c"]
    S, N, Hq, Hkv, D, ps = c["slots"], int(s["n"].max()), c["Hq"], c["Hkv"], c["D"], c["page"]
    G = Hq // Hkv
    L = int((s["length_now"] + s["n"]).max())
    pages = s["table"][:, : -(-L // ps)].clamp(min=0).long()
    k = s["k"][0][pages].transpose(1, 2).reshape(S, Hkv, -1, D)[:, :, :L].float()
    q = s["q"].new_zeros(S, N, Hq, D, dtype=torch.float32)
    q[s["slot"], s["at"]] = s["q"].float()
    q = q.view(S, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, N * G, D)
    scores = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D))
    del k
    mask = s["mask"].new_zeros(S, N)
    mask[s["slot"], s["at"]] = s["mask"]
    place = torch.arange(L, device=DEV)[None, :] - s["length"][:, None]
    node = place[:, None, :]
    seen = (node < 0) | ((node < 64) & ((mask[:, :, None] >> node.clamp(0, 63)) & 1).bool())
    scores.view(S, Hkv, N, G, L).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    z = p.sum(dim=3, keepdim=True)
    v = s["v"][0][pages].transpose(1, 2).reshape(S, Hkv, -1, D)[:, :, :L].float()
    v.masked_fill_((place >= torch.from_numpy(s["n"]).to(DEV)[:, None])[:, None, :, None], 0.0)
    out = torch.where(z > 0, (p @ v) / z, 0.0)
    lse = (top + torch.log(z)).view(S, Hkv, N, G).transpose(1, 2).reshape(S, N, Hq)[s["slot"], s["at"]]
    out = out.view(S, Hkv, N, G, D).transpose(1, 2).reshape(S, N, Hq, D)[s["slot"], s["at"]]
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _rotated(x, weight, cos, sin, pairs, rot):
    """x / sqrt(mean x^2 + eps) * weight, then the first `rot` values of each head turned pair by pair"""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(dim=2, keepdim=True) + 1e-6) * weight
    h = rot // 2
    a, b = (x[:, :, :h], x[:, :, h:rot]) if pairs == "halves" else (x[:, :, 0:rot:2], x[:, :, 1:rot:2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(turned, dim=2) if pairs == "halves" else torch.stack(turned, dim=3).flatten(2)
    return torch.cat([turned, x[:, :, rot:]], dim=2)


def _append(s):
    c = s["c"]
    angle = s["pos"].double()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotated(s["q_in"], s["q_weight"], cos, sin, c["pairs"], c["rot"]).to(s["q_in"].dtype)
    k = _rotated(s["k_in"], s["k_weight"], cos, sin, c["pairs"], c["rot"]).to(s["k_in"].dtype)
    place = s["length"][s["slot"]].long() + s["at"]
    page = s["table"][s["slot"], place // c["page"]].long()
    s["k"][0][page, :, place % c["page"]] = k
    s["v"][0][page, :, place % c["page"]] = s["v_in"]
    return {"q": q, "k": s["k"], "v": s["v"]}


def _reserve(table, used, ref, length, extra, ps):
    """pages for `extra` more tokens of every slot: the lowest free ones, slot after slot"""
    need = (-(-(length + extra) // ps) - used).clamp(min=0).long()
    end = need.cumsum(0)
    total = int(end[-1])
    free = (ref == 0).nonzero()[:total, 0]
    slot = torch.repeat_interleave(torch.arange(len(need), device=DEV), need)
    table[slot, used[slot] + torch.arange(total, device=DEV) - (end - need)[slot]] = free.int()
    ref[free] = 1
    used += need.int()


def _step(s):
    """room for the drafted nodes; the kept nodes' keys and values moved together; pages past the last kept one given back"""
    ps = s["c"]["page"]
    table, used, ref, length = s["table"], s["used"], s["ref"], s["length"]
    _reserve(table, used, ref, length, s["extra"], ps)
    kept, path = s["kept"], s["path"].long()
    i = torch.arange(path.shape[1], device=DEV)
    slot, i = (i[None, :] < kept[:, None]).nonzero(as_tuple=True)
    frm, to = length[slot].long() + path[slot, i], length[slot].long() + i
    frm_page, to_page = table[slot, frm // ps].long(), table[slot, to // ps].long()
    s["k"][:, to_page, :, to % ps] = s["k"][:, frm_page, :, frm % ps]
    s["v"][:, to_page, :, to % ps] = s["v"][:, frm_page, :, frm % ps]
    torch.add(length, kept, out=s["length_out"])
    left = -(-s["length_out"] // ps)
    at = torch.arange(table.shape[1], device=DEV)[None, :]
    gone = (at >= left[:, None]) & (at < used[:, None])
    pages = table[gone].long()
    ref.index_put_((pages,), torch.full_like(pages, -1, dtype=torch.int32), accumulate=True)
    table.masked_fill_(gone, -1)
    torch.minimum(used, left, out=used)
    return {"k": s["k"], "v": s["v"], "table": table, "used": used, "ref": ref, "length": s["length_out"]}


def _fork(s):
    """the copies' pages given back; then each copy shares its parent's full pages and gets a page with the rest of the last one"""
    ps = s["c"]["page"]
    table, used, ref, length, parent = s["table"], s["used"], s["ref"], s["length"], s["parent"]
    copies = (s["which"] != 0).nonzero()[:, 0]
    at = torch.arange(table.shape[1], device=DEV)[None, :]
    pages = table[copies][at < used[copies, None]].long()
    ref.index_put_((pages,), torch.full_like(pages, -1, dtype=torch.int32), accumulate=True)
    table[copies], used[copies], length[copies] = -1, 0, 0
    frm = parent[copies].long()
    n = length[frm]
    full, rest = n // ps, n % ps
    table[copies] = torch.where(at < full[:, None], table[frm], -1)
    pages = table[copies][at < full[:, None]].long()
    ref.index_put_((pages,), torch.ones_like(pages, dtype=torch.int32), accumulate=True)
    used[copies], length[copies] = full, n
    extra = torch.zeros_like(used)
    extra[copies] = (rest > 0).int()
    _reserve(table, used, ref, used * ps, extra, ps)
    which, t = (torch.arange(ps, device=DEV)[None, :] < rest[:, None]).nonzero(as_tuple=True)
    last = full[which].long()
    old, new = table[frm[which], last].long(), table[copies[which], last].long()
    s["k"][:, new, :, t] = s["k"][:, old, :, t]
    s["v"][:, new, :, t] = s["v"][:, old, :, t]
    return {"k": s["k"], "v": s["v"], "table": table, "used": used, "ref": ref, "length": length}


def _accept(s):
    """from the root on: the first child whose draft is the token chosen at the node, until there is none"""
    off, n = s["off"].long(), torch.from_numpy(s["n"]).to(DEV)
    S, N = len(n), s["c"]["nodes"]
    at = torch.arange(N, device=DEV)
    here = at[None, :] < n[:, None]
    flat = torch.where(here, off[:-1, None] + at, 0)
    token, draft = s["token"][flat], s["draft"][flat]
    parent = torch.where(here & (at > 0), s["parent"][flat].long(), -1)
    child = (parent[:, None, :] == at[None, :, None]) & (draft[:, None, :] == token[:, :, None])  # [slot, node, its child]
    first = child & (child.cumsum(2) == 1)
    # which nodes are reached: steps along `first`, doubled six times (2^6 >= 64)
    reach = first.float() + torch.eye(N, device=DEV)
    r2 = (reach @ reach).clamp_(max=1)
    r4 = (r2 @ r2).clamp_(max=1)
    r8 = (r4 @ r4).clamp_(max=1)
    r16 = (r8 @ r8).clamp_(max=1)
    r32 = (r16 @ r16).clamp_(max=1)
    on = ((r32 @ r32)[:, 0] > 0) & here
    kept = on.sum(1)
    place = torch.where(on, on.cumsum(1) - 1, N)
    path = torch.full((S, N + 1), -1, dtype=torch.int32, device=DEV)
    path.scatter_(1, place, at.int().expand(S, N))
    path[:, N] = -1
    last = path.gather(1, (kept - 1)[:, None]).long()
    return {"accepted": (kept - 1).int(), "kept": kept.int(), "next": token.gather(1, last)[:, 0], "path": path[:, :N].contiguous()}


def run(state):
    s = state
    c = s["c"]
    kind = c["kind"]
    if own:
        import arcinfer_b200 as ab

        if kind == "attention":
            got = ab.tree_attention(s["q"], s["cache"], s["off"], c["nodes"], mask=s["mask"], want_lse=True)
            return {"out": got["out"], "lse": got["lse"]}
        if kind == "append":
            q = ab.cache_append(s["cache"], s["q_in"], s["k_in"], s["v_in"], s["off"], s["pos"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                                interleaved=c["pairs"] == "neighbours")
            return {"q": q, "k": s["k"], "v": s["v"]}
        if kind == "accept":
            got = ab.accept_tree(s["token"], s["draft"], s["parent"], s["off"], c["nodes"])
            return {"accepted": got["accepted"], "kept": got["kept"], "next": got["next"], "path": got["path"]}
        if kind == "step":
            ab.cache_reserve(s["cache"], s["extra"])
            ab.cache_compact(s["cache"], s["kept"], s["path"], length_out=s["length_out"])
        else:
            ab.cache_free(s["cache"], s["which"])
            ab.cache_fork(s["cache"], s["parent"])
        return {"k": s["k"], "v": s["v"], "table": s["table"], "used": s["used"], "ref": s["ref"], "length": s["length_out"] if kind == "step" else s["length"]}
    return {"attention": _attention, "append": _append, "step": _step, "fork": _fork, "accept": _accept}[kind](s)


def work(case):
    """What a pass cannot do without: every cached key and value that is attended to read once, queries
    in and results out, the moved or copied rows once each way, the lists of pages."""
    c = case
    kind = c["kind"]
    if kind == "accept":
        n = _spread(c["slots"], c["nodes"], 0.5 if c["slots"] > 1 else 0.0, 1)
        return {"bytes": int(12 * n.sum() + 4 * c["slots"] * (4 + c["nodes"])), "flops": 0}
    row = c["Hkv"] * c["D"] * 2
    if kind == "fork":
        copies = c["parents"] * c["children"]
        pages = c["ctx"] // c["page"] + 1
        return {"bytes": copies * (c["rest"] * row * 2 * 2 * c["layers"] + pages * 4 * 6), "flops": 0}
    n = _nodes(c)
    if kind == "step":
        return {"bytes": c["slots"] * ((c["kept"] - 1) * row * 2 * 2 * c["layers"] + 64), "flops": 0}
    if kind == "append":
        return {"bytes": int(n.sum()) * 2 * (c["Hq"] + 2 * c["Hkv"]) * c["D"] * 2, "flops": int(n.sum()) * (c["Hq"] + c["Hkv"]) * c["D"] * 7}
    length = _lengths(c)
    pages = int((-(-(length + n) // c["page"])).sum())
    return {"bytes": int((length + n).sum()) * row * 2 + pages * 4 + int(n.sum()) * c["Hq"] * (c["D"] * 4 + 4), "flops": int((n * (length + n / 4)).sum()) * c["Hq"] * c["D"] * 4}


def exact(case, seed):
    """The computed numbers from the formulas in 64 bits, slot by slot and token by token's place; what
    is moved or counted has no such value."""
    kind = case["kind"]
    if kind not in ("attention", "append"):
        return None
    s = prepare(case, seed)
    c, off = case, s["off"].tolist()
    D, ps, Hq, Hkv = c["D"], c["page"], c["Hq"], c["Hkv"]
    table = s["table"].long()
    if kind == "append":
        angles = np.outer(s["pos"].cpu().numpy().astype(np.float64), s["inv_freq"].cpu().numpy())
        turn = torch.from_numpy(np.exp(1j * angles)).to(DEV)[:, None, :]
        done = {}
        for name in ("q", "k"):
            x, w, rot = s[name + "_in"].double(), s[name + "_weight"], c["rot"]
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
            pairs = x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if c["pairs"] == "halves" else x[..., :rot].unflatten(-1, (rot // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            done[name] = torch.cat([(z.transpose(-1, -2) if c["pairs"] == "halves" else z).flatten(-2), x[..., rot:]], dim=-1)
        k, v = s["k"].double(), s["v"].double()
        for r in range(c["slots"]):
            a, b = off[r], off[r + 1]
            place = int(s["length"][r]) + torch.arange(b - a, device=DEV)
            page = table[r][place // ps]
            for h in range(Hkv):
                k[0, page, h, place % ps] = done["k"][a:b, h]
                v[0, page, h, place % ps] = s["v_in"][a:b, h].double()
        return {"q": done["q"], "k": k, "v": v}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(c["slots"]):
        a, b, n = off[r], off[r + 1], int(s["length"][r])
        place = torch.arange(n + b - a, device=DEV)
        page = table[r][place // ps]
        allowed = torch.ones(b - a, n + b - a, dtype=torch.bool, device=DEV)
        for i, bits in enumerate(s["mask"][a:b].tolist()):
            allowed[i, n:] = torch.tensor([bool((bits >> j) & 1) for j in range(b - a)], device=DEV)
        for h in range(Hkv):
            k, v = (s[x][0, page, h, place % ps].double() for x in ("k", "v"))
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                x = (s["q"][a:b, i].double() @ k.T) / math.sqrt(D)
                x = torch.where(allowed, x, -math.inf)
                lse[a:b, i] = torch.logsumexp(x, dim=1)
                out[a:b, i] = torch.exp(x - lse[a:b, i, None]) @ v
    return {"out": out, "lse": lse}
