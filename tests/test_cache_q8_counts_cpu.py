"""Counts of attention over the 8-bit cache next to 32 bits: what a loop would step over is refused before any launch."""
from ctypes import byref, c_void_p

import pytest

import test_cache_q8_cpu as base
from nanoflow_b200 import ops


# (requests, query heads, KV heads, page list): products from 2^31 - 65536 on, which steps of up to 148 * 16 warps would pass
@pytest.mark.parametrize("requests,heads,kv_heads,indices", [
    (0x7ffffff0, 1, 1, 4), (0x7fff0001, 1, 1, 4), (0x7ffffff0 // 8, 8, 2, 4), (0x7fff8000 // 16, 16, 1, 4), (3, 8, 2, 0x7ffffff0 // 2), (3, 1, 1, 0x7ffffff0)])
def test_counts_without_room_for_a_step_are_refused(requests, heads, kv_heads, indices):
    p = base._attn(req_count=requests, q_heads=heads, kv_heads=kv_heads, num_indices=indices)
    assert ops.lib().nfk_attn_decode_q8(byref(p), c_void_p(0)) == 1
