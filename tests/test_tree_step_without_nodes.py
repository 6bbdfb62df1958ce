"""A step in which no slot has nodes: every call of it is accepted, and says so."""
import numpy as np
import pytest
import torch

import arcinfer_b200 as ab

P = 1 << 20  # an aligned address that is never read


@pytest.mark.skipif(torch.cuda.is_available(), reason="would be launched with addresses that are not there")
def test_the_walk_takes_no_rows():
    """(without a device the launch fails; the arguments are not what is refused)"""
    assert ab.lib.arcs_accept_tree(None, None, None, P, 3, 0, 8, P, P, P, P, 8, None, None) != 1
    for i in range(3):
        lists = [P, P, P]
        lists[i] = None
        assert ab.lib.arcs_accept_tree(*lists, P, 3, 1, 8, P, P, P, P, 8, None, None) == 1


@pytest.mark.gpu
def test_a_step_without_nodes():
    import kvutil as kv

    S, page = 3, 16
    cache, _ = kv.make_cache(1, [20, 0, 16], [0] * S, heads=2, page=page, dim=64)
    before = [x.clone() for x in (cache.table, cache.used, cache.ref, cache.length)]
    off, parent, depth, mask = ab.tree_lists([[]] * S)
    off, none = kv.i32(off), kv.i32(parent)
    ab.cache_reserve(cache, kv.i32([0] * S))
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = ab.cache_append(cache, x, x, x, off, none, torch.zeros(32, dtype=torch.float64, device="cuda"))
    out = ab.tree_attention(q, cache, off, 8, mask=torch.from_numpy(mask).cuda(), want_lse=True)
    assert out["out"].shape == (0, 2, 64) and out["lse"].shape == (0, 2)
    acc = ab.accept_tree(none, none, none, off, 8, status=cache.status)
    ab.cache_compact(cache, acc["kept"], acc["path"])
    torch.cuda.synchronize()
    assert int(cache.status.item()) == 0
    assert acc["accepted"].tolist() == [-1] * S and acc["kept"].tolist() == [0] * S and acc["next"].tolist() == [-1] * S and (acc["path"] == -1).all()
    for a, b in zip(before, (cache.table, cache.used, cache.ref, cache.length)):
        assert torch.equal(a, b)
    # rows that are announced but not there
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    acc = ab.accept_tree(none, none, none, kv.i32(np.array([0, 2, 2, 2])), 8, status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 9 and acc["kept"].tolist() == [0] * S
