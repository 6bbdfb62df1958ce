"""The largest scales of the attention (no device needed: one that is taken is refused for its workspace, which is looked at afterwards)."""
import ctypes as C
import math

import pytest

import arcinfer_b200 as ab
from arcinfer_b200 import kvcache as kvc

P = 1 << 20  # an aligned address that is never read


@pytest.mark.parametrize("scale,status", [(1e-30, 3), (1.0, 3), (2.3e38, 3), (2.4e38, 1), (2.9e38, 1), (3.4e38, 1)])
def test_scale_times_log2_e_is_a_number(scale, status):
    """the kernels hold scale * log2 e in 32 bits: infinite, it would make NaN of a score of zero"""
    assert (scale / math.log(2) < 2.0**128) == (status == 3)
    c = kvc.CacheArgs(k=P, v=P, dtype=1, layers=1, n_pages=4, page_size=16, heads=1, dim=64, layer_stride=0, page_stride=1024, head_stride=1024, token_stride=64, slots=1, max_pages=4, table=P,
                      used=P, ref=P, len=P, status=None)  # fmt: skip
    a = kvc.TreeAttentionArgs(cache=C.addressof(c), layer=0, T=4, Hq=1, q=P, q_token_stride=64, q_head_stride=64, out=P, out_token_stride=64, out_head_stride=64, node_off=P, max_nodes=4, scale=scale,
                              workspace=P, workspace_bytes=16)  # fmt: skip
    assert ab.lib.arcs_tree_attention(C.byref(a), None) == status
