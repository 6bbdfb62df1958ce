"""Nodes whose values are infinite or no numbers, in batches of many short texts: every CTA of the attention
works on one item after the other, and each item's values belong to its own rows."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _check(got, want, size, top, dtype):
    """The same NaN and infinities, and the bound of kvutil.check_attention for the numbers: half a step of the result, half
    a step and 2^-16 of sum weight * |value|, and weights among fp16's subnormal numbers (`top`: the largest finite value,
    150 places at most)."""
    import kvutil as kv

    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    far = torch.isinf(want)
    assert torch.equal(torch.isinf(got), far) and torch.equal(got[far], want[far])
    fin = torch.isfinite(want)
    u = kv.HALF_STEP[dtype]
    bound = u * want.abs() + (u + 2.0**-16) * size + kv.SMALLEST[dtype] * (1 + 150 * 2.0**-7 * top)
    assert ((got - want).abs()[fin] <= bound[fin]).all(), ((got - want).abs() / bound)[fin].max().item()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,Hq,most", [(64, 8, 6), (64, 64, 20), (128, 16, 6), (128, 64, 20), (256, 16, 6), (256, 64, 4)])
def test_every_item_shows_its_own(dim, Hq, most, dtype):
    """320 slots x 8 key heads, one tile of keys and some with two; (64 and 128, 64 heads) two tiles of rows an item at
    most, most items with fewer than 32 rows"""
    import arcinfer_b200 as ab
    import kvutil as kv

    g = np.random.default_rng(dim + Hq)
    slots, heads, page, dt = 320, 8, 16, kv.DTYPES[dtype]
    lens = [int(x) for x in g.integers(0, 121, slots)]
    nodes = [int(x) for x in g.integers(1, 5, slots)]
    nodes[5] = nodes[200] = most
    for s in range(0, slots, 9):
        lens[s] = 126  # nodes on both sides of a tile's end
    cache, rows = kv.make_cache(dim + Hq, lens, nodes, heads, page, dim, dt)
    off, parent, depth, mask = ab.tree_lists([kv.random_parents(g, n, 3) for n in nodes])
    gen = torch.Generator(device="cuda")
    gen.manual_seed(dim)
    q = torch.randn(int(off[-1]), Hq, dim, generator=gen, device="cuda").to(dt)
    # in two thirds of the slots: bad values in some nodes, at each one's own columns
    table = cache.table.cpu().numpy()
    for s in range(slots):
        if s % 3 == 0:
            continue
        for j in range(nodes[s]):
            if j and g.random() < 0.4:
                continue
            place, c = lens[s] + j, int(g.integers(0, dim - 2))
            bad = torch.tensor([[math.inf, -math.inf, math.nan][int(x)] for x in g.integers(0, 3, 2)], dtype=dt, device="cuda")
            cache.v[0, int(table[s, place // page]), :, place % page, c : c + 2] = bad
            rows[s][1][0, :, place, c : c + 2] = bad
    want, size, top = [], [], 0.0
    for s in range(slots):
        a, b = int(off[s]), int(off[s + 1])
        v = rows[s][1][0]
        w, _, z = kv.attention64(q[a:b], rows[s][0][0], v, lens[s], [int(m) & (2**64 - 1) for m in mask[a:b]], dim**-0.5)
        want.append(w), size.append(z)
        top = max(top, v[torch.isfinite(v)].abs().max().item())
    want, size = torch.cat(want), torch.cat(size)
    assert torch.isnan(want).any() and torch.isinf(want).any() and torch.isfinite(want).any()
    o, m = kv.i32(off), torch.from_numpy(mask).cuda()
    for _ in range(20):
        got = ab.tree_attention(q, cache, o, most, mask=m)["out"]
        torch.cuda.synchronize()
        assert int(cache.status.item()) == 0
        _check(got, want, size, top, dt)
