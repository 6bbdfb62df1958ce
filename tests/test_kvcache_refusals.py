"""Calls over the paged cache that are refused before anything is launched (no device needed), and the host's lists of trees."""
import ctypes as C

import numpy as np
import pytest
import torch

import arcinfer_b200 as ab
from arcinfer_b200 import kvcache as kvc

P = 1 << 20  # an aligned address that is never read


def _cache(**kw):
    f = dict(k=P, v=P, dtype=1, layers=2, n_pages=8, page_size=16, heads=2, dim=64, layer_stride=8 * 2048, page_stride=2048, head_stride=1024, token_stride=64, slots=3, max_pages=4,
             table=P, used=P, ref=P, len=P, status=None)  # fmt: skip
    f.update(kw)
    return kvc.CacheArgs(**f)


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(used=None), dict(len=None), dict(dtype=0), dict(dtype=3), dict(layers=0), dict(n_pages=0), dict(page_size=8), dict(page_size=48),
              dict(page_size=512), dict(heads=0), dict(heads=2000), dict(dim=96), dict(dim=512), dict(layer_stride=4), dict(page_stride=2044), dict(head_stride=32), dict(token_stride=60),
              dict(token_stride=-64), dict(slots=0), dict(slots=4097), dict(max_pages=0), dict(max_pages=1 << 28), dict(k=P + 8), dict(v=P + 2)]  # fmt: skip


def _append(c, **kw):
    f = dict(cache=C.addressof(c), layer=0, T=4, Hq=4, q=P, k=P, v=P, q_stride=256, k_stride=128, v_stride=128, q_out=P, q_out_stride=256, eps=1e-6, rot=64, inv_freq=P, pos=P, node_off=P)
    f.update(kw)
    return kvc.AppendArgs(**f)


def _attention(c, **kw):
    f = dict(cache=C.addressof(c), layer=0, T=4, Hq=4, q=P, q_token_stride=256, q_head_stride=64, out=P, out_token_stride=256, out_head_stride=64, node_off=P, max_nodes=8, scale=0.125, workspace=P,
             workspace_bytes=1 << 40)
    f.update(kw)
    return kvc.TreeAttentionArgs(**f)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_cache(bad):
    c = _cache(**bad)
    p = C.addressof(c)
    for call in (lambda: ab.lib.arcs_cache_reserve(p, P, None), lambda: ab.lib.arcs_cache_fork(p, P, P, None), lambda: ab.lib.arcs_cache_free(p, P, None),
                 lambda: ab.lib.arcs_cache_compact(p, P, P, 4, P, None), lambda: ab.lib.arcs_cache_append(C.byref(_append(c)), None),
                 lambda: ab.lib.arcs_tree_attention(C.byref(_attention(c)), None)):  # fmt: skip
        assert call() == 1
        assert b"cache" in ab.lib.arcs_last_error()


def test_lists():
    c = _cache()
    p = C.addressof(c)
    assert ab.lib.arcs_cache_reserve(p, None, None) == 1 and ab.lib.arcs_cache_reserve(None, P, None) == 1
    assert ab.lib.arcs_cache_fork(p, None, P, None) == 1 and ab.lib.arcs_cache_fork(p, P, None, None) == 1
    assert ab.lib.arcs_cache_free(p, None, None) == 1
    for a in ((None, P, 4, P), (P, None, 4, P), (P, P, 0, P), (P, P, 4, None)):
        assert ab.lib.arcs_cache_compact(p, *a, None) == 1
    no_ref = _cache(ref=None)
    assert ab.lib.arcs_cache_reserve(C.addressof(no_ref), P, None) == 1
    assert ab.lib.arcs_cache_compact(C.addressof(no_ref), P, P, 4, P, None) == 1


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(T=-1), dict(Hq=0), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(pos=None), dict(node_off=None),
                                 dict(inv_freq=None), dict(rot=8), dict(rot=80), dict(rot=-16), dict(q_stride=252), dict(q_stride=128), dict(k_stride=64), dict(v_stride=64),
                                 dict(q_out_stride=128), dict(q=P + 8), dict(k=P + 4), dict(v=P + 2), dict(q_out=P + 8), dict(q_weight=P + 4), dict(k_weight=P + 8), dict(eps=-1.0), dict(eps=float("nan"))], ids=str)  # fmt: skip
def test_append(bad):
    c = _cache()
    assert ab.lib.arcs_cache_append(C.byref(_append(c, **bad)), None) == 1
    assert b"cache_append" in ab.lib.arcs_last_error()


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(T=-1), dict(Hq=0), dict(Hq=3), dict(Hq=130), dict(q=None), dict(out=None), dict(node_off=None), dict(max_nodes=0),
                                 dict(max_nodes=65), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_token_stride=252), dict(q_head_stride=32),
                                 dict(out_token_stride=0), dict(out_head_stride=60), dict(q=P + 8), dict(out=P + 4)], ids=str)  # fmt: skip
def test_attention(bad):
    c = _cache()
    assert ab.lib.arcs_tree_attention(C.byref(_attention(c, **bad)), None) == 1
    assert b"tree_attention" in ab.lib.arcs_last_error()


def test_attention_workspace():
    c = _cache()
    need = ab.lib.arcs_tree_attention_workspace_bytes(3, 2, 4, 64, 8)
    assert need > 0
    for bad in (dict(workspace=None), dict(workspace_bytes=need - 1)):
        assert ab.lib.arcs_tree_attention(C.byref(_attention(c, **bad)), None) == 3
    for sizes in ((0, 2, 4, 64, 8), (3, 0, 4, 64, 8), (3, 2, 3, 64, 8), (3, 2, 4, 96, 8), (3, 2, 4, 64, 0), (3, 2, 4, 64, 65)):
        assert ab.lib.arcs_tree_attention_workspace_bytes(*sizes) == 0


def test_accept_tree():
    ok = [P, P, P, P, 3, 10, 8, P, P, P, P, 8, None, None]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, 0), (5, -1), (6, 0), (6, 65), (7, None), (8, None), (9, None), (10, None), (11, 7)):
        a = list(ok)
        a[i] = v
        assert ab.lib.arcs_accept_tree(*a) == 1
        assert b"accept_tree" in ab.lib.arcs_last_error()


def test_nothing_to_do_needs_no_device():
    c = _cache()
    assert ab.lib.arcs_cache_append(C.byref(_append(c, T=0)), None) == 0
    assert ab.lib.arcs_tree_attention(C.byref(_attention(c, T=0)), None) == 0


def _host_cache():
    z = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(2, 8, 2, 16, 64, dtype=torch.bfloat16)
    return ab.KVCache(k, k.clone(), z(3, 4), z(3), z(8), z(3))


def test_binding_refuses_tensors_of_another_kind(monkeypatch):
    c = _host_cache()
    z = lambda *n, dtype=torch.int32: torch.zeros(*n, dtype=dtype)  # noqa: E731
    q, k = z(4, 4, 64, dtype=torch.bfloat16), z(4, 2, 64, dtype=torch.bfloat16)
    inv = z(32, dtype=torch.float64)
    launched = []
    for name in ("arcs_cache_reserve", "arcs_cache_fork", "arcs_cache_free", "arcs_cache_compact", "arcs_cache_append", "arcs_tree_attention", "arcs_accept_tree"):
        monkeypatch.setattr(kvc.lib, name, lambda *a: launched.append(a) or 0)
    bad = [
        lambda: ab.KVCache(c.k, c.v.float(), c.table, c.used, c.ref, c.length), lambda: ab.KVCache(c.k.float(), c.v.float(), c.table, c.used, c.ref, c.length),
        lambda: ab.KVCache(c.k, c.v.transpose(2, 3).contiguous().transpose(2, 3), c.table, c.used, c.ref, c.length), lambda: ab.KVCache(c.k, c.v, c.table.long(), c.used, c.ref, c.length),
        lambda: ab.KVCache(c.k, c.v, c.table, z(4), c.ref, c.length), lambda: ab.KVCache(c.k, c.v, c.table, c.used, z(7), c.length), lambda: ab.KVCache(c.k, c.v, c.table[0], c.used, c.ref, c.length),
        lambda: ab.cache_reserve(c, z(2)), lambda: ab.cache_reserve(c, z(3, dtype=torch.int64)), lambda: ab.cache_fork(c, z(6)[::2]), lambda: ab.cache_free(c, z(4)),
        lambda: ab.cache_compact(c, z(3), z(3)), lambda: ab.cache_compact(c, z(3), z(2, 4)), lambda: ab.cache_compact(c, z(3), z(3, 4), length_out=z(2)),
        lambda: ab.cache_append(c, q, k, k, z(3), z(4), inv), lambda: ab.cache_append(c, q, k, k, z(4), z(3), inv), lambda: ab.cache_append(c, q, k[:3], k, z(4), z(4), inv),
        lambda: ab.cache_append(c, q, k, k, z(4), z(4), inv.float()), lambda: ab.cache_append(c, q.half(), k, k, z(4), z(4), inv),
        lambda: ab.cache_append(c, q, k, k, z(4), z(4), inv, q_weight=z(64, dtype=torch.bfloat16)), lambda: ab.cache_append(c, q[:, ::2], k, k, z(4), z(4), inv),
        lambda: ab.tree_attention(q.half(), c, z(4), 8), lambda: ab.tree_attention(q[:, :, :32], c, z(4), 8), lambda: ab.tree_attention(q, c, z(4), 8, mask=z(4)),
        lambda: ab.tree_attention(q, c, z(3), 8), lambda: ab.tree_attention(q, c, z(4), 8, out=q[:3]), lambda: ab.accept_tree(z(4), z(3), z(4), z(2), 4),
        lambda: ab.accept_tree(z(4).long(), z(4), z(4), z(2), 4),
    ]  # fmt: skip
    for i, call in enumerate(bad):
        with pytest.raises(ab.ArcsError):
            call()
        assert not launched, i


def test_tensors_on_the_host_are_refused(monkeypatch):
    c = _host_cache()
    z = lambda *n, dtype=torch.int32: torch.zeros(*n, dtype=dtype)  # noqa: E731
    q, k = z(4, 4, 64, dtype=torch.bfloat16), z(4, 2, 64, dtype=torch.bfloat16)
    launched = []
    for name in ("arcs_cache_reserve", "arcs_cache_fork", "arcs_cache_free", "arcs_cache_compact", "arcs_cache_append", "arcs_tree_attention", "arcs_accept_tree"):
        monkeypatch.setattr(kvc.lib, name, lambda *a: launched.append(a) or 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    for call in (lambda: ab.cache_reserve(c, z(3)), lambda: ab.cache_fork(c, z(3)), lambda: ab.cache_free(c, z(3)), lambda: ab.cache_compact(c, z(3), z(3, 4)),
                 lambda: ab.cache_append(c, q, k, k, z(4), z(4), z(32, dtype=torch.float64)), lambda: ab.tree_attention(q, c, z(4), 8), lambda: ab.accept_tree(z(4), z(4), z(4), z(2), 4)):  # fmt: skip
        with pytest.raises(ValueError):
            call()
        assert not launched


def test_tree_lists():
    off, parent, depth, mask = ab.tree_lists([[-1, 0, 0, 1, 3], [], [-1]])
    assert off.tolist() == [0, 5, 5, 6] and parent.tolist() == [-1, 0, 0, 1, 3, -1] and depth.tolist() == [0, 1, 1, 2, 3, 0]
    assert mask.tolist() == [1, 0b11, 0b101, 0b1011, 0b11011, 1]
    chain = ab.tree_lists([[-1] + list(range(63))])[3]
    assert chain.view(np.uint64)[-1] == np.uint64(2**64 - 1)
    for bad in ([-1, 1], [0], [-1, -1], [-1, 0, 5], [-1] + [0] * 64):
        with pytest.raises(ab.ArcsError):
            ab.tree_lists([bad])


def test_calls_run_on_the_device_of_the_cache(monkeypatch):
    """with another device current, the cache's is made current for the launch, and its stream is used"""
    seen, current = [], [0]

    class Device:
        def __init__(self, dev):
            self.index = dev.index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *a):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    for index in (0, 1, 0):
        kvc._enqueue(torch.device("cuda", index), lambda *a: seen.append((current[-1],) + a) or 0, "call", 5)
    assert seen == [(0, 5, 100), (1, 5, 101), (0, 5, 100)] and current == [0]
    with pytest.raises(ab.ArcsError, match="call"):
        kvc._enqueue(torch.device("cuda", 1), lambda *a: 4, "call")
