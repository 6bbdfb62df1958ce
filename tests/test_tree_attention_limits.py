"""Sizes of a cache up to which the attention counts its work, on both sides of the limit (no device needed: a call that is
within it is refused for its workspace, which is looked at afterwards)."""
import ctypes as C

import pytest

import arcinfer_b200 as ab
from arcinfer_b200 import kvcache as kvc

P = 1 << 20  # an aligned address that is never read


def _status(slots, heads, Hq, dim, max_nodes, max_pages, page_stride=None):
    """of a call over tables of max_pages pages of 256 tokens, with too small a workspace"""
    c = kvc.CacheArgs(k=P, v=P, dtype=1, layers=1, n_pages=64, page_size=256, heads=heads, dim=dim, layer_stride=0, page_stride=page_stride or heads * 256 * dim, head_stride=256 * dim, token_stride=dim,
                      slots=slots, max_pages=max_pages, table=P, used=P, ref=P, len=P, status=None)  # fmt: skip
    a = kvc.TreeAttentionArgs(cache=C.addressof(c), layer=0, T=4, Hq=Hq, q=P, q_token_stride=Hq * dim, q_head_stride=dim, out=P, out_token_stride=Hq * dim, out_head_stride=dim, node_off=P,
                              max_nodes=max_nodes, scale=0.125, workspace=P, workspace_bytes=16)  # fmt: skip
    return ab.lib.arcs_tree_attention(C.byref(a), None)


# slots x heads x blocks x (c x tiles of 128 places + e) < 2^31. With more than 128 rows a key head at dim 64 and 128: c = 6, e = 18 and
# blocks of 256 rows; else c = 1, e = 4 and blocks of 128
@pytest.mark.parametrize("heads,Hq,dim,max_nodes,most", [
    (8, 16, 128, 8, 32765),   # 32768 items x (65530 + 4)
    (8, 16, 64, 64, 32765),   # 128 rows
    (8, 64, 256, 64, 8189),   # 512 rows, four blocks: 131072 x (16378 + 4)
    (8, 64, 128, 64, 2729),   # 512 rows, two blocks: 65536 x (5458 x 6 + 18)
    (8, 64, 64, 32, 5459),    # 256 rows, one block: 32768 x (10918 x 6 + 18)
])  # fmt: skip
def test_units_of_work(heads, Hq, dim, max_nodes, most):
    for max_pages, status in ((most, 3), (most + 1, 1)):
        assert _status(4096, heads, Hq, dim, max_nodes, max_pages) == status
    assert b"too large" in ab.lib.arcs_last_error()
    # the kernel for other strides counts nothing
    assert _status(4096, heads, Hq, dim, max_nodes, most + 1, page_stride=heads * 256 * dim + 8) == 3
