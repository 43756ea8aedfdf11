"""Attention behind a shared prefix for numbers of rows (requests x heads) that are no multiple of a CTA's four."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import test_cache_q8_gpu as base
from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref


# so many rows that the last CTA starts when the first one has ended; few rows, and a budget that makes few CTAs walk over them
@pytest.mark.parametrize("requests,heads,kv_heads,ctas", [(3001, 7, 1, 0), (3002, 9, 3, 0), (4003, 5, 5, 0), (234, 7, 1, 400), (234, 7, 1, 100), (401, 3, 3, 1)])
def test_the_first_row_is_written_once(requests, heads, kv_heads, ctas):
    own = [i % 4 for i in range(requests)]
    pages = sum(-(-x // 16) for x in own) + 4
    pool, scale = base._cache(pages, kv_heads, 64, torch.int8)
    ptr, idx, last = base._lists(own, pages - 4, 5)
    front = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")
    q = torch.randn(requests, heads * 64, device="cuda").to(torch.bfloat16)
    args = (pool, scale, torch.arange(requests + 1, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=requests, q_heads=heads, kv_heads=kv_heads, head_dim=64, prefix_len=50)
    want = ref.attn_decode_q8(q, *args, q_heads=heads, req_begin=0, req_count=requests, prefix_pages=front, prefix_len=50)
    for _ in range(3):
        out = torch.full_like(q, 3.0)
        ops.attn_decode_shared_q8(q, out, *args, front, 50, q_heads=heads, req_begin=0, req_count=requests, workspace=ws, num_ctas=ctas)
        base._check_rows(out, want, 64)
