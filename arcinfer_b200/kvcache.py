"""The paged cache and the verification of a tree of drafts over it (include/arcsample.h): pages
reserved, forked, freed and compacted, keys and values brought there, a tree's attention, and the walk
that accepts a path. Tensors are torch CUDA tensors; every call enqueues on torch's current stream of
the cache's device and returns without synchronising."""
import ctypes as C
import math
import struct

import numpy as np
import torch

from .capi import ArcsError, _check, _stream, lib

F16, BF16 = 2, 1
TREE_MAX = 64
_CODES = {torch.bfloat16: BF16, torch.float16: F16}


class CacheArgs(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("layers", C.c_int32), ("n_pages", C.c_int32),
        ("page_size", C.c_int32), ("heads", C.c_int32), ("dim", C.c_int32),
        ("layer_stride", C.c_int64), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("token_stride", C.c_int64),
        ("slots", C.c_int32), ("max_pages", C.c_int32),
        ("table", C.c_void_p), ("used", C.c_void_p), ("ref", C.c_void_p), ("len", C.c_void_p), ("status", C.c_void_p),
    ]  # fmt: skip


class AppendArgs(C.Structure):
    _fields_ = [
        ("cache", C.c_void_p), ("layer", C.c_int32), ("T", C.c_int32), ("Hq", C.c_int32),
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p),
        ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
        ("q_out", C.c_void_p), ("q_out_stride", C.c_int64), ("q_weight", C.c_void_p), ("k_weight", C.c_void_p),
        ("eps", C.c_float), ("rot", C.c_int32), ("interleaved", C.c_int32),
        ("inv_freq", C.c_void_p), ("pos", C.c_void_p), ("node_off", C.c_void_p),
    ]  # fmt: skip


class TreeAttentionArgs(C.Structure):
    _fields_ = [
        ("cache", C.c_void_p), ("layer", C.c_int32), ("T", C.c_int32), ("Hq", C.c_int32),
        ("q", C.c_void_p), ("q_token_stride", C.c_int64), ("q_head_stride", C.c_int64),
        ("out", C.c_void_p), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
        ("lse", C.c_void_p), ("node_off", C.c_void_p), ("mask", C.c_void_p), ("max_nodes", C.c_int32), ("scale", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]  # fmt: skip


lib.arcs_cache_reserve.restype = C.c_int
lib.arcs_cache_reserve.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
lib.arcs_cache_fork.restype = C.c_int
lib.arcs_cache_fork.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
lib.arcs_cache_free.restype = C.c_int
lib.arcs_cache_free.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
lib.arcs_cache_compact.restype = C.c_int
lib.arcs_cache_compact.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]
lib.arcs_cache_append.restype = C.c_int
lib.arcs_cache_append.argtypes = [C.c_void_p, C.c_void_p]
lib.arcs_tree_attention_workspace_bytes.restype = C.c_size_t
lib.arcs_tree_attention_workspace_bytes.argtypes = [C.c_int32] * 5
lib.arcs_tree_attention.restype = C.c_int
lib.arcs_tree_attention.argtypes = [C.c_void_p, C.c_void_p]
lib.arcs_accept_tree.restype = C.c_int
lib.arcs_accept_tree.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p, C.c_void_p, C.c_void_p,
                                 C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p]  # fmt: skip


# The argument blocks of the calls of a step, packed (a ctypes structure filled field by field takes three times as
# long, which a small batch notices); native alignment is the compiler's.
_append_block = struct.Struct("@P3i4x3P3qPq2Pf2i4x3P")
_attention_block = struct.Struct("@P3i4xP2qP2q3PifPN")
assert _append_block.size == C.sizeof(AppendArgs) and _attention_block.size == C.sizeof(TreeAttentionArgs)
_i32, _i64, _f32, _f64 = torch.int32, torch.int64, torch.float32, torch.float64
_empty = torch.empty


def _list(name, t, dtype, n, dev):
    """a contiguous device list of n (None: any number of) values"""
    if t.dtype is dtype and t.device == dev and t.is_contiguous() and (n is None or t.numel() == n):
        return t.data_ptr()
    raise ArcsError(f"{name} must be a contiguous {dtype} tensor{'' if n is None else f' of {n} values'} on {dev}, not {t.dtype} {tuple(t.shape)} on {t.device}")


def _enqueue(dev, fn, what, *args):
    """launches on the current stream of the device, with that device current"""
    stream = _stream(dev)
    if dev.index is None or dev.index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _check(rc, what)


class KVCache:
    """Pools, lists and sizes of a paged cache (arcs_cache). k, v: [layers, pages, heads, page_size,
    dim] bfloat16 or float16 (or without the layers), any strides that leave a row's values side by
    side, the same for both. table int32 [slots, max_pages], used / length int32 [slots], ref int32
    [pages]: see include/arcsample.h. The tensors are held, not copied: they are the cache's state.
    status: int32 [1], 0 or the first arcs_status that a kernel raised."""

    def __init__(self, k, v, table, used, ref, length, status=None):
        k, v = (x.unsqueeze(0) if x.dim() == 4 else x for x in (k, v))
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.stride(4) != 1 or k.dtype != v.dtype or k.dtype not in _CODES or k.device != v.device:
            raise ArcsError("k and v must be bfloat16 or float16 [layers, pages, heads, page_size, dim] with the same strides, a row's values side by side")
        dev = k.device
        layers, n_pages, heads, page_size, dim = k.shape
        if table.dim() != 2:
            raise ArcsError("table must be [slots, max_pages]")
        slots, max_pages = table.shape
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=dev)
        i32 = torch.int32
        self.device, self.slots, self.heads, self.dim, self.dtype, self.layers = dev, slots, heads, dim, k.dtype, layers
        self.k, self.v, self.table, self.used, self.ref, self.length, self.status = k, v, table, used, ref, length, status
        self.args = CacheArgs(k.data_ptr(), v.data_ptr(), _CODES[k.dtype], layers, n_pages, page_size, heads, dim, k.stride(0), k.stride(1), k.stride(2), k.stride(3),
                              slots, max_pages, _list("table", table, i32, None, dev), _list("used", used, i32, slots, dev), _list("ref", ref, i32, n_pages, dev),
                              _list("length", length, i32, slots, dev), _list("status", status, i32, 1, dev))
        self.ptr = C.addressof(self.args)
        self.workspace_bytes = {}
        self.scale = 1.0 / math.sqrt(dim)

    @staticmethod
    def empty(layers, n_pages, heads, page_size, dim, slots, max_pages, dtype=torch.bfloat16, device="cuda"):
        """a cache of zeros, all pages free"""
        pool = lambda: torch.zeros(layers, n_pages, heads, page_size, dim, dtype=dtype, device=device)  # noqa: E731
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=device)  # noqa: E731
        return KVCache(pool(), pool(), z(slots, max_pages) - 1, z(slots), z(n_pages), z(slots))


def cache_reserve(cache, extra):
    """arcs_cache_reserve: pages for extra[s] (int32 [slots]) more tokens behind every slot's length."""
    _enqueue(cache.device, lib.arcs_cache_reserve, "arcs_cache_reserve", cache.ptr, _list("extra", extra, torch.int32, cache.slots, cache.device))


def cache_fork(cache, parent):
    """arcs_cache_fork: slot s becomes a copy of slot parent[s] (int32 [slots], -1: nothing). Returns
    int32 [slots], 1 where a copy was made."""
    done = torch.empty(cache.slots, dtype=torch.int32, device=cache.device)
    _enqueue(cache.device, lib.arcs_cache_fork, "arcs_cache_fork", cache.ptr, _list("parent", parent, torch.int32, cache.slots, cache.device), done.data_ptr())
    return done


def cache_free(cache, which):
    """arcs_cache_free: every slot with which[s] != 0 (int32 [slots]) gives its pages back."""
    _enqueue(cache.device, lib.arcs_cache_free, "arcs_cache_free", cache.ptr, _list("which", which, torch.int32, cache.slots, cache.device))


def cache_compact(cache, kept, path, length_out=None):
    """arcs_cache_compact: the kept[s] nodes path[s, :kept[s]] (int32 [slots], [slots, n], as accept_tree
    returns them) become the slot's next tokens. length_out: int32 [slots] for the new lengths; without
    it they replace the cache's."""
    dev = cache.device
    if path.dim() != 2 or path.shape[0] != cache.slots:
        raise ArcsError(f"path must be [{cache.slots}, n]")
    out = cache.length if length_out is None else length_out
    _enqueue(cache.device, lib.arcs_cache_compact, "arcs_cache_compact", cache.ptr, _list("kept", kept, torch.int32, cache.slots, dev), _list("path", path, torch.int32, None, dev),
          path.shape[1], _list("length_out", out, torch.int32, cache.slots, dev))
    return out


def _heads(name, t, T, H, dim, dtype, dev):
    """[T, H, dim] of the cache's type, a row's heads side by side: (address, row stride)"""
    if t.shape == (T, H, dim) and t.dtype is dtype and t.device == dev:
        row, head, one = t.stride()
        if one == 1 and (head == dim or H == 1):
            return t.data_ptr(), row if T > 1 else max(row, H * dim)
    raise ArcsError(f"{name} must be {dtype} [{T}, {H}, {dim}] on {dev} with a row's heads side by side, not {t.dtype} {tuple(t.shape)}")


def cache_append(cache, q, k, v, node_off, pos, inv_freq, layer=0, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, q_out=None):
    """arcs_cache_append: norm (where a float32 weight [dim] is given) and rotation of the step's queries
    [T, Hq, dim] and keys [T, heads, dim], head by head; keys and values [T, heads, dim] go to the cache.
    pos: int32 [T]; inv_freq: float64 [rot / 2]; node_off: int32 [slots + 1]. Returns the queries (q_out,
    which may be q itself, or a new tensor)."""
    if q.dim() != 3:
        raise ArcsError("q must be [T, Hq, dim]")
    dev, dtype, heads, dim = cache.device, cache.dtype, cache.heads, cache.dim
    T, Hq, _ = q.shape
    if q_out is None:
        q_out = _empty((T, Hq, dim), dtype=dtype, device=dev)
        op, os_ = q_out.data_ptr(), Hq * dim
    else:
        op, os_ = _heads("q_out", q_out, T, Hq, dim, dtype, dev)
    qp, qs = _heads("q", q, T, Hq, dim, dtype, dev)
    kp, ks = _heads("k", k, T, heads, dim, dtype, dev)
    vp, vs = _heads("v", v, T, heads, dim, dtype, dev)
    block = _append_block.pack(
        cache.ptr, layer, T, Hq, qp, kp, vp, qs, ks, vs, op, os_, 0 if q_weight is None else _list("q_weight", q_weight, _f32, dim, dev),
        0 if k_weight is None else _list("k_weight", k_weight, _f32, dim, dev), eps, 2 * inv_freq.numel(), int(interleaved), _list("inv_freq", inv_freq, _f64, None, dev),
        _list("pos", pos, _i32, T, dev), _list("node_off", node_off, _i32, cache.slots + 1, dev))  # fmt: skip
    _enqueue(dev, lib.arcs_cache_append, "arcs_cache_append", block)
    return q_out


def tree_attention(q, cache, node_off, max_nodes, mask=None, layer=0, scale=None, want_lse=False, out=None):
    """arcs_tree_attention: q [T, Hq, dim] of the cache's type; node_off int32 [slots + 1]; mask int64 [T]
    (bit j of a row: it sees node j of its slot) or None for chains; max_nodes: no slot has more nodes.
    scale: 1 / sqrt(dim) unless given. Returns a dict: out (like q, or the tensor given) and, with
    want_lse, lse float32 [T, Hq]."""
    dev, dim = cache.device, cache.dim
    if q.dim() != 3 or q.dtype is not cache.dtype or q.device != dev:
        raise ArcsError(f"q must be {cache.dtype} [T, Hq, {dim}] on {dev}")
    T, Hq, d = q.shape
    qt, qh, one = q.stride()
    if d != dim or one != 1:
        raise ArcsError(f"q must be [T, Hq, {dim}], a head's values side by side")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else _empty((T, Hq, dim), dtype=cache.dtype, device=dev)
        ot, oh = Hq * dim, dim
    else:
        if out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1:
            raise ArcsError("out must be like q")
        ot, oh, _ = out.stride()
    r = {"out": out}
    lse = 0
    if want_lse:
        r["lse"] = x = _empty((T, Hq), dtype=_f32, device=dev)
        lse = x.data_ptr()
    nbytes = cache.workspace_bytes.get((Hq, max_nodes))
    if nbytes is None:
        nbytes = cache.workspace_bytes[Hq, max_nodes] = lib.arcs_tree_attention_workspace_bytes(cache.slots, cache.heads, Hq, dim, max_nodes)
    # (new for every call, from torch's allocator: calls on two streams, or in two graphs, never share one)
    ws = _empty(nbytes, dtype=torch.uint8, device=dev)
    if T < 2 or Hq < 2:  # (a single row's or a single head's stride is of no meaning, but looked at)
        qt, ot = (x if T > 1 else max(x, dim) // 8 * 8 for x in (qt, ot))
        qh, oh = (x if Hq > 1 else max(x, dim) // 8 * 8 for x in (qh, oh))
    block = _attention_block.pack(
        cache.ptr, layer, T, Hq, q.data_ptr(), qt, qh, out.data_ptr(), ot, oh, lse, _list("node_off", node_off, _i32, cache.slots + 1, dev),
        0 if mask is None else _list("mask", mask, _i64, T, dev), max_nodes, cache.scale if scale is None else scale, ws.data_ptr(), nbytes)  # fmt: skip
    _enqueue(dev, lib.arcs_tree_attention, "arcs_tree_attention", block)
    return r


def accept_tree(token, draft, parent, node_off, max_nodes, status=None):
    """arcs_accept_tree: token, draft, parent int32 [T], node_off int32 [slots + 1]. Returns a dict of
    int32 tensors: accepted, kept, next [slots], path [slots, max_nodes]. status: int32 [1], optional."""
    dev = token.device
    T, slots = token.numel(), node_off.numel() - 1
    args = (_list("token", token, _i32, None, dev), _list("draft", draft, _i32, T, dev), _list("parent", parent, _i32, T, dev), _list("node_off", node_off, _i32, None, dev))
    accepted = _empty(slots, dtype=_i32, device=dev)
    kept, last = torch.empty_like(accepted), torch.empty_like(accepted)
    path = _empty((slots, max_nodes), dtype=_i32, device=dev)
    _enqueue(dev, lib.arcs_accept_tree, "arcs_accept_tree", *args, slots, T, max_nodes, accepted.data_ptr(), kept.data_ptr(), last.data_ptr(), path.data_ptr(), max_nodes,
             None if status is None else _list("status", status, _i32, 1, dev))
    return {"accepted": accepted, "kept": kept, "next": last, "path": path}


def tree_lists(parents):
    """What the calls want to know of a step's trees, from one list of parents' indices per slot (the
    root first, its parent -1; a parent before its children): node_off int32 [slots + 1], parent int32
    [T], depth int32 [T] (a node's position is its slot's length plus this), mask int64 [T] (a node
    sees its ancestors and itself), as numpy arrays."""
    off, parent, depth, mask = [0], [], [], []
    for tree in parents:
        if len(tree) > TREE_MAX:
            raise ArcsError(f"a tree has {len(tree)} nodes: {TREE_MAX} at most")
        d, m = [], []
        for i, p in enumerate(tree):
            p = int(p)
            if (i == 0) != (p == -1) or p >= i or p < -1:
                raise ArcsError(f"node {i}'s parent is {p}: the root's is -1, any other's comes before it")
            d.append(0 if i == 0 else d[p] + 1)
            m.append((1 << i) | (0 if i == 0 else m[p]))
        off.append(off[-1] + len(tree))
        parent += [int(p) for p in tree]
        depth += d
        mask += m
    return (np.asarray(off, np.int32), np.asarray(parent, np.int32), np.asarray(depth, np.int32), np.asarray(mask, np.uint64).view(np.int64))
