"""The CTA budget of attention over the 8-bit cache holds for every kernel of a call: grids are read from captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import test_cache_q8_gpu as base
from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref


def _grids(call):
    """Numbers of CTAs of the kernels that `call` launches."""
    from cuda.bindings import driver as cu

    def ok(answer):
        assert answer[0] == cu.CUresult.CUDA_SUCCESS, answer[0]
        return answer[1:]

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = cu.CUgraph(init_value=graph.raw_cuda_graph())
    nodes, count = ok(cu.cuGraphGetNodes(raw))
    nodes, count = ok(cu.cuGraphGetNodes(raw, count))
    grids = []
    for node in nodes[:count]:
        if ok(cu.cuGraphNodeGetType(node))[0] == cu.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            of = ok(cu.cuGraphKernelNodeGetParams(node))[0]
            grids.append(of.gridDimX * of.gridDimY * of.gridDimZ)
    return grids


# the joins of many rows by ranges of one head and of two, of few rows, of many rows behind a prefix, of few
@pytest.mark.parametrize("heads,kv_heads,lengths,prefix", [
    (8, 2, [37 * i % 301 for i in range(1, 200)], 0), (16, 2, [37 * i % 301 for i in range(1, 120)], 0), (8, 2, [4000, 7, 333, 0, 50], 0),
    (8, 2, [11 * i % 40 for i in range(200)], 700), (8, 2, [100, 0, 5], 700), (8, 2, [9], 0)])
@pytest.mark.parametrize("ctas", [0, 1, 3, 20, 131])
def test_no_kernel_has_more_blocks_than_the_budget(heads, kv_heads, lengths, prefix, ctas):
    n = len(lengths)
    pages = sum(-(-x // 16) for x in lengths) + -(-prefix // 16) + 1
    pool, scale = base._cache(pages, kv_heads, 128, torch.int8)
    ptr, idx, last = base._lists(lengths, pages, 3)
    front = torch.arange(-(-prefix // 16), dtype=torch.int32, device="cuda")
    q = torch.randn(n, heads * 128, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 3.0)
    args = (pool, scale, torch.arange(n + 1, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=n, q_heads=heads, kv_heads=kv_heads, head_dim=128, prefix_len=prefix)
    st = ops.new_status()

    def call():
        ops.attn_decode_shared_q8(q, out, *args, front, prefix, q_heads=heads, req_begin=0, req_count=n, workspace=ws, num_ctas=ctas, status=st)

    call()
    ops.check_status(st)
    base._check_rows(out, ref.attn_decode_q8(q, *args, q_heads=heads, req_begin=0, req_count=n, prefix_pages=front if prefix else None,
                                             prefix_len=prefix), 128)
    grids = _grids(call)
    assert grids and (ctas == 0 or max(grids) <= ctas), grids
