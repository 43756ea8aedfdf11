"""Rows that a call of attention over the 8-bit cache must write, and those that it must not, where the output held something else before."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import test_cache_q8_gpu as base
from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref

HEADS, KV_HEADS, DIM, PREFIX = 8, 2, 128, 40
# a batch in one launch, one whose states are joined row by row, one whose states are joined by ranges
BATCHES = {"few": [100, 7, 333], "rows": [4000, 7, 333, 0, 50], "ranges": [37 * i % 301 for i in range(1, 200)]}


class Case:
    def __init__(self, lengths, kind=torch.float8_e4m3fn):
        self.n = len(lengths)
        self.pages = sum(-(-x // 16) for x in lengths) + 5
        self.pool, self.scale = base._cache(self.pages, KV_HEADS, DIM, kind)
        self.ptr, self.idx, self.last = base._lists(lengths, self.pages, 3)
        self.qo = torch.arange(self.n + 1, dtype=torch.int32, device="cuda")
        self.q = torch.randn(self.n, HEADS * DIM, device="cuda").to(torch.bfloat16)
        self.front = base._i32([4, 0, 2])
        self.ws = ops.decode_workspace_q8(requests=self.n, q_heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, prefix_len=PREFIX)
        self.st = ops.new_status()

    def run(self, shared, reported=False, **change):
        """The rows of a call on an output of 3s."""
        a = {**dict(qo=self.qo, ptr=self.ptr, idx=self.idx, last=self.last, front=self.front), **change}
        out = torch.full_like(self.q, 3.0)
        kw = dict(q_heads=HEADS, req_begin=0, req_count=self.n, workspace=self.ws, status=self.st)
        if shared:
            ops.attn_decode_shared_q8(self.q, out, self.pool, self.scale, a["qo"], a["ptr"], a["idx"], a["last"], a["front"], PREFIX, **kw)
        else:
            ops.attn_decode_q8(self.q, out, self.pool, self.scale, a["qo"], a["ptr"], a["idx"], a["last"], **kw)
        if reported:
            with pytest.raises(RuntimeError, match="out-of-range"):
                ops.check_status(self.st)
        else:
            ops.check_status(self.st)
        return out

    def want(self, shared, **change):
        a = {**dict(qo=self.qo, ptr=self.ptr, idx=self.idx, last=self.last), **change}
        return ref.attn_decode_q8(self.q, self.pool, self.scale, a["qo"], a["ptr"], a["idx"], a["last"], q_heads=HEADS, req_begin=0, req_count=self.n,
                                  prefix_pages=self.front if shared else None, prefix_len=PREFIX if shared else 0)


ALL = [pytest.mark.parametrize("batch", list(BATCHES)), pytest.mark.parametrize("shared", [False, True], ids=["plain", "shared"])]


def every(test):
    for mark in ALL:
        test = mark(test)
    return test


@every
def test_every_call_writes_its_rows(batch, shared):
    c = Case(BATCHES[batch])
    want = c.want(shared)
    for _ in range(3):
        base._check_rows(c.run(shared), want, DIM)


@every
@pytest.mark.parametrize("page", ["negative", "beyond"])
def test_a_page_that_does_not_exist_spoils_one_request(batch, shared, page):
    c = Case(BATCHES[batch])
    at = int(c.ptr[2])                            # the first page of request 2
    idx = c.idx.clone()
    idx[at] = -5 if page == "negative" else c.pages
    out, want = c.run(shared, True, idx=idx), c.want(shared)
    assert bool(out[2].isfinite().all()) and not bool((out[2] == 3).all())
    del want[2]
    base._check_rows(out, want, DIM)


@every
@pytest.mark.parametrize("row", [-1, "beyond"])
def test_a_row_that_does_not_exist_is_left_out(batch, shared, row):
    c = Case(BATCHES[batch])
    qo = c.qo.clone()
    qo[1] = c.n if row == "beyond" else row
    out, want = c.run(shared, True, qo=qo), c.want(shared)
    assert bool((out[1] == 3).all())
    del want[1]
    base._check_rows(out, want, DIM)


@every
@pytest.mark.parametrize("how", ["falls", "ends behind the pages", "begins below them"])
def test_lists_that_are_none_are_as_if_there_were_no_pages(batch, shared, how):
    """Exact zeros, or what the prefix alone gives."""
    c = Case(BATCHES[batch])
    ptr = c.ptr.clone()
    if how == "falls":
        ptr[2] = ptr[1] - 1
    elif how == "begins below them":
        ptr[0] = -3
    else:
        ptr[c.n] += 7
    out = c.run(shared, True, ptr=ptr)
    if not shared:
        assert not out.any()
        return
    base._check_rows(out, c.want(True, ptr=torch.zeros_like(c.ptr), last=torch.zeros_like(c.last)), DIM)


@pytest.mark.parametrize("batch", list(BATCHES))
def test_a_page_of_the_prefix_that_does_not_exist(batch):
    """Reported; every row is written."""
    c = Case(BATCHES[batch])
    out = c.run(True, True, front=base._i32([1, 2, c.pages]))
    assert bool(out.isfinite().all()) and not bool((out == 3).all(1).any())
    base._check_rows(c.run(True), c.want(True), DIM)
