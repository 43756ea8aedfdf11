"""The 8-bit KV cache against plain forms in 64 bits: the write into it, its pages as bf16, attention over it.

Tolerances count the roundings. Half a step is 2^-8 of the value for bf16, 2^-4 for e4m3 (2^-10 of the unit for its smallest
numbers), half a unit for whole numbers, 2^-11 for the f16 weights of the second product; fp32 sums of up to 128 products of exact
factors are off by less than 128 * 2^-24 of the sum of magnitudes.
"""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = pytest.mark.parametrize("kind", [E4M3, INT8], ids=["e4m3", "int8"])


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lists(lengths, pages, seed, extra=0):
    """indptr, indices, last page lengths of requests of these lengths over a pool of `pages`, `extra` entries behind them."""
    counts = [-(-n // 16) for n in lengths]
    ptr = [0]
    for c in counts:
        ptr.append(ptr[-1] + c)
    assert ptr[-1] <= pages
    order = random.Random(seed).sample(range(pages), ptr[-1])
    return _i32(ptr), _i32(order + [10 ** 6] * extra), _i32([n - 16 * (c - 1) if c else 0 for n, c in zip(lengths, counts)])


def _cache(pages, kv_heads, dim, kind, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(pages, 2, kv_heads, 16, dim, device="cuda", generator=g)
    x *= torch.exp(spread * torch.randn(pages, 2, kv_heads, 16, 1, device="cuda", generator=g))
    scale = (x.abs().amax(-1) / ref.Q8_LARGEST[kind]).contiguous()
    y = x / scale[..., None]
    return (y.round() if kind == INT8 else y.clamp(-448, 448)).to(kind), scale


def _raw(pool):
    return pool.view(torch.int8)


# ---- the write ---------------------------------------------------------------------------------------------------------
def _append_case(T, heads, kv_heads, dim, kind, norm, table, far, pad, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    new = [1] * T if T < 5 else [T - 3 - T // 2, 1, T // 2, 2]
    past = [r.randint(0, far) for _ in new]
    counts = [(p + n + 15) // 16 for p, n in zip(past, new)]
    first = [sum(counts[:i]) for i in range(len(counts) + 1)]
    used = sorted({first[b] + (p + i) // 16 for b, (p, n) in enumerate(zip(past, new)) for i in range(n)})
    pages = len(used) + 3
    indices = [0] * first[-1]
    for u, page in zip(used, r.sample(range(pages), len(used))):
        indices[u] = page
    width = (heads + 2 * kv_heads) * dim
    wide = torch.randn(T, width + pad, device="cuda", generator=g).to(torch.bfloat16)
    wide *= 10.0 ** r.randint(-3, 3)
    qkv = wide[:, pad // 2:pad // 2 + width]
    norms = [(1 + 0.1 * torch.randn(dim, device="cuda", generator=g)).to(torch.bfloat16) if norm else None for _ in range(2)]
    pool, scale = _cache(pages, kv_heads, dim, kind, seed)
    return dict(qkv=qkv, pool=pool, scale=scale, norms=norms, new=new, past=past, first=first, indices=indices,
                positions=_i32([p + i for p, n in zip(past, new) for i in range(n)]),
                req=_i32([b for b, n in enumerate(new) for _ in range(n)]),
                inv=(500000.0 ** (-torch.arange(0, dim, 2, device="cuda").double() / dim)).float(), table=table)


@KINDS
@pytest.mark.parametrize("T,heads,kv_heads,dim,norm,table,far,pad", [
    (1, 32, 8, 128, True, False, 100000, 0), (3, 64, 8, 128, False, False, 2 ** 24, 0), (37, 28, 4, 128, True, False, 700, 64),
    (37, 9, 3, 64, True, True, 700, 16), (700, 32, 8, 128, False, True, 50, 0), (130, 12, 12, 64, False, False, 3000, 8),
    (130, 12, 12, 64, False, False, 3000, 48),
    (5, 1, 1, 64, True, False, 0, 0), (1500, 16, 1, 128, True, False, 20, 0)])
def test_append(kind, T, heads, kv_heads, dim, norm, table, far, pad):
    c = _append_case(T, heads, kv_heads, dim, kind, norm, table, far, pad)
    off = dict(q_heads=heads, kv_heads=kv_heads, head_dim=dim, q_off=2 * kv_heads * dim, k_off=0, v_off=kv_heads * dim)
    before, scale_before = _raw(c["pool"]).clone(), c["scale"].clone()
    q = torch.full((T, heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    st = ops.new_status()
    cos_sin = ops.rope_table(c["inv"], c["positions"]) if table else None
    if pad // 2 % 8:                              # rows that do not start on 16 bytes are refused
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.rope_append_q8(c["qkv"], q, c["pool"], c["scale"], c["inv"], c["positions"], c["req"], _i32(c["first"]), _i32(c["indices"]), **off)
        return
    ops.rope_append_q8(c["qkv"], q, c["pool"], c["scale"], c["inv"], c["positions"], c["req"], _i32(c["first"]), _i32(c["indices"]), **off,
                       q_norm=c["norms"][0], k_norm=c["norms"][1], eps=1e-6, cos_sin=cos_sin, status=st)
    ops.check_status(st)
    cpu = lambda t: None if t is None else t.cpu()
    rq, rk, rv = ref.rope_append_q8(c["qkv"].cpu(), c["inv"].cpu(), c["positions"].cpu(), **off, q_norm=cpu(c["norms"][0]),
                                    k_norm=cpu(c["norms"][1]), eps=1e-6)
    # fp32 sums, factors and angles: 2^-20 of the vector's largest entry; a table holds angles that are off by 2^-24 of the
    # position's (and its own cosine and sine by as much again)
    angle = 2.0 ** -23 * float(c["positions"].max()) if table else 0.0
    noise = lambda y: y.abs().amax(-1, keepdim=True) * (2.0 ** -20 + 2 * angle)
    err = (q.cpu().double().view_as(rq) - rq).abs()
    assert bool((err <= 2.0 ** -8 * rq.abs() + noise(rq)).all()), float(err.max())
    page = _i32(c["indices"])[(_i32(c["first"])[c["req"].long()] + c["positions"] // 16).long()].long()
    slot = (c["positions"] % 16).long()
    numbers, scale = c["pool"].view(torch.int8)[page, :, :, slot].cpu().view(kind).double(), c["scale"][page, :, :, slot].cpu().double()
    for side, y in ((0, rk), (1, rv)):
        n, s = numbers[:, side], scale[:, side]
        most = y.abs().amax(-1)
        slack = noise(y) if side == 0 else most[..., None] * 2.0 ** -20
        assert bool(((s * ref.Q8_LARGEST[kind] - most).abs() <= 2.0 ** -22 * most + slack[..., 0]).all())
        half = 0.5 * s[..., None] if kind == INT8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s[..., None])
        err = (n * s[..., None] - y).abs()
        assert bool((err <= half + 2 * slack).all()), float((err / s[..., None]).max())
        assert float(n.abs().max()) <= ref.Q8_LARGEST[kind]
    # what was not written is as it was
    mask = torch.zeros(c["pool"].shape[0], 16, dtype=torch.bool, device="cuda")
    mask[page, slot] = True
    keep = ~mask[:, None, None, :].expand_as(c["scale"])
    assert torch.equal(_raw(c["pool"])[keep], before[keep]) and torch.equal(c["scale"][keep], scale_before[keep])


@KINDS
def test_append_of_odd_vectors(kind):
    """Zeros, tiny and huge vectors, infinities and NaN, one to a token; a page list that is too short, pages that do not exist."""
    dim, T = 128, 9
    x = torch.randn(T, 3 * dim, device="cuda").to(torch.bfloat16)
    x[0] = 0
    x[1] *= 2.0 ** -100
    x[2] *= 2.0 ** 120
    x[3, dim + 5] = float("inf")                 # the value's row
    x[4, dim + 5] = float("nan")
    x[5] *= 2.0 ** -70
    pool, scale = _cache(4, 1, dim, kind)
    _raw(pool).fill_(3)
    scale.fill_(5.0)
    st = ops.new_status()
    # tokens 6, 7 and 8: a position behind the list, a page that does not exist, a request that does not exist
    req, pos = _i32([0, 0, 0, 0, 0, 0, 0, 1, 7]), _i32([0, 1, 2, 3, 4, 5, 16, 0, 0])
    q = torch.zeros(T, dim, dtype=torch.bfloat16, device="cuda")
    ops.rope_append_q8(x, q, pool, scale, torch.ones(dim // 2, device="cuda"), pos, req, _i32([0, 1, 2]), _i32([2, 4]), q_heads=1, kv_heads=1,
                       head_dim=dim, q_off=2 * dim, k_off=0, v_off=dim, status=st)
    with pytest.raises(RuntimeError, match="out-of-range"):
        ops.check_status(st)
    v, vs = pool[2, 1, 0].double(), scale[2, 1, 0]
    assert vs[0] == 0 and vs[1] == 0 and not v[:2].any()
    assert bool(vs[3:5].isnan().all()) and not v[3:5].any()
    for t in (2, 5):
        y = x[t, dim:2 * dim].double()
        half = 0.5 * vs[t].double() if kind == INT8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * vs[t].double())
        assert bool(((v[t] * vs[t].double() - y).abs() <= half + 2.0 ** -19 * y.abs().max()).all())
    assert bool((_raw(pool)[[0, 1, 3]] == 3).all()) and bool((scale[[0, 1, 3]] == 5).all())
    assert bool((_raw(pool)[2, :, :, 6:] == 3).all()) and bool((scale[2, :, :, 6:] == 5).all())
    assert bool(q[:6].isfinite().all()) and bool(q[6:].any())


# ---- pages as bf16 -----------------------------------------------------------------------------------------------------
@KINDS
@pytest.mark.parametrize("pages,listed,kv_heads,dim", [(1, 1, 1, 64), (40, 37, 4, 64), (9, 5, 3, 128), (300, 257, 8, 128), (7, 0, 2, 128)])
def test_read(kind, pages, listed, kv_heads, dim):
    pool, scale = _cache(pages, kv_heads, dim, kind)
    ids = random.Random(1).sample(range(pages), listed)
    if listed > 2:
        ids[1] = ids[0]
    out = ops.kv_read_q8(pool, scale, _i32(ids))
    want = ref.kv_values_q8(pool, scale, _i32(ids))
    assert out.shape == want.shape
    # the product is rounded to fp32 and then to bf16
    assert bool(((out.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.abs()).all())


def test_read_of_every_number():
    for kind in (E4M3, INT8):
        pool = torch.arange(256, device="cuda").to(torch.uint8).view(torch.int8).repeat(2 * 16 * 64 // 256).view(1, 2, 1, 16, 64)
        scale = torch.ones(1, 2, 1, 16, device="cuda")
        scale[0, 0, 0, 4:8] = float("nan")
        out = ops.kv_read_q8(pool.view(kind), scale, _i32([0])).float()
        want = pool.view(kind).float() * scale[..., None]
        assert torch.equal(out.nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))      # exact: eight bits fit bf16


def test_read_leaves_places_of_missing_pages():
    pool, scale = _cache(3, 2, 64, INT8)
    out = torch.full((3, 2, 2, 16, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    st = ops.new_status()
    ops.kv_read_q8(pool, scale, _i32([1, 3, -1]), out=out, status=st)
    with pytest.raises(RuntimeError, match="out-of-range"):
        ops.check_status(st)
    assert bool((out[1:] == 9).all()) and not bool((out[0] == 9).all())


# ---- attention ---------------------------------------------------------------------------------------------------------
def _check_rows(out, want, head_dim):
    for row, (o, size, score, most) in want.items():
        got = out[row].double().cpu().view(o.shape)
        assert bool(got.isfinite().all())
        # weights 2^-11, exponentials 2^-20, the scores' sums twice; the result 2^-8.
        # A weight is p * 2^7 * scale / v_ref in f16, with v_ref at most twice the largest scale, and below 2^-14 it is rounded to a
        # multiple of 2^-24: off by 2^-25 at most, which is 2^-25 * 2^-7 * 2 = 2^-31 of the largest scale; times a number, 2^-31 of
        # the largest |v|, for each token. The sum that this is divided by is at least 1: the largest score has p >= 1, since the
        # reference is a score that was seen (and a piece's share of the joined result is at most 1).
        tol = 2.0 ** -8 * o.abs() + size * (2.0 ** -11 + 2.0 ** -19 + 2 * score * 2.0 ** -17) + 2.0 ** -31 * most + 1e-30
        err = (got - o).abs()
        assert bool((err <= tol).all()), (row, float((err / tol).max()), float(err.max()))


LENGTHS = {
    "one": [1], "none": [0, 0], "edges": [15, 16, 17, 0, 1, 31, 32, 33, 0], "mixed": [333, 4000, 1, 700, 0, 16, 2500, 63],
    "long": [20000], "short": [1 + 7 * i % 60 for i in range(300)], "even": [256] * 40}


@KINDS
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (7, 1, 128), (16, 1, 128), (4, 4, 64), (9, 3, 64), (22, 2, 64)])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_decode(kind, heads, kv_heads, dim, lengths):
    n = LENGTHS[lengths]
    pages = sum(-(-x // 16) for x in n) + 3
    pool, scale = _cache(pages, kv_heads, dim, kind)
    ptr, idx, last = _lists(n, pages, 5, extra=4)
    rows = torch.randperm(len(n) + 2)[:len(n)]
    qo = _i32(rows.tolist() + [0])
    q = torch.randn(len(n) + 2, heads * dim, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 3.0)
    ws = ops.decode_workspace_q8(requests=len(n), q_heads=heads, kv_heads=kv_heads, head_dim=dim)
    st = ops.new_status()
    for _ in range(2):                            # the workspace is ready again
        ops.attn_decode_q8(q, out, pool, scale, qo, ptr, idx, last, q_heads=heads, req_begin=0, req_count=len(n), workspace=ws, status=st)
        ops.check_status(st)
        _check_rows(out, ref.attn_decode_q8(q, pool, scale, qo, ptr, idx, last, q_heads=heads, req_begin=0, req_count=len(n)), dim)
    other = [r for r in range(len(n) + 2) if r not in rows.tolist()]
    assert bool((out[other] == 3).all())


@pytest.mark.parametrize("ctas", [1, 3, 37])
def test_decode_part_of_the_batch_with_few_ctas(ctas):
    n = [40, 500, 3, 0, 77, 16, 900, 5]
    pool, scale = _cache(120, 2, 128, E4M3)
    ptr, idx, last = _lists(n, 120, 3)
    q = torch.randn(8, 8 * 128, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 3.0)
    ws = ops.decode_workspace_q8(requests=8, q_heads=8, kv_heads=2, head_dim=128, prefix_len=100)
    qo = torch.arange(9, dtype=torch.int32, device="cuda")
    args = (pool, scale, qo, ptr, idx, last)
    ops.attn_decode_q8(q, out, *args, q_heads=8, req_begin=2, req_count=5, workspace=ws, sm_scale=0.2, num_ctas=ctas)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=8, req_begin=2, req_count=5, sm_scale=0.2), 128)
    assert bool((out[:2] == 3).all()) and bool((out[7:] == 3).all())
    out.fill_(3.0)
    ops.attn_decode_shared_q8(q, out, *args, idx[:7].flip(0).contiguous(), 100, q_heads=8, req_begin=2, req_count=5, workspace=ws, sm_scale=0.2,
                              num_ctas=ctas)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=8, req_begin=2, req_count=5, sm_scale=0.2, prefix_pages=idx[:7].flip(0), prefix_len=100), 128)
    assert bool((out[:2] == 3).all()) and bool((out[7:] == 3).all())


@KINDS
@pytest.mark.parametrize("shared", [0, 70])
def test_what_lies_behind_a_request_is_never_seen(kind, shared):
    """NaN, infinities and NaN numbers in the places of tokens that there are none of; a NaN that is seen stays in its request."""
    n = [5, 40, 17, 300]
    pool, scale = _cache(60, 2, 128, kind)
    ptr, idx, last = _lists(n, 50, 3)
    front = _i32(list(set(range(60)) - set(idx.tolist()))[:-(-shared // 16) or 1])
    q = torch.randn(4, 8 * 128, device="cuda").to(torch.bfloat16)
    ends = [(int(idx[int(ptr[b + 1]) - 1]), int(last[b])) for b in range(4)] + ([(int(front[-1]), (shared - 1) % 16 + 1)] if shared else [])
    for page, used in ends:
        scale[page, :, :, used:] = float("nan")
        scale[page, 0, :, used + 1::2] = float("inf")
        _raw(pool)[page, :, :, used:] = 0x7f
    args = (pool, scale, torch.arange(5, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=4, q_heads=8, kv_heads=2, head_dim=128, prefix_len=shared)
    out = torch.empty_like(q)

    def run():
        if shared:
            ops.attn_decode_shared_q8(q, out, *args, front, shared, q_heads=8, req_begin=0, req_count=4, workspace=ws)
        else:
            ops.attn_decode_q8(q, out, *args, q_heads=8, req_begin=0, req_count=4, workspace=ws)

    run()
    want = ref.attn_decode_q8(q, *args, q_heads=8, req_begin=0, req_count=4, prefix_pages=front, prefix_len=shared)
    _check_rows(out, want, 128)
    scale[int(idx[int(ptr[1])]), 1, 0, 3] = float("nan")         # a value of request 1, KV head 0
    run()
    assert bool(out[1, :4 * 128].isnan().all())
    out[1, :4 * 128] = 0
    want[1][0][:4] = 0
    _check_rows(out, want, 128)


@KINDS
def test_scores_and_scales_of_any_size(kind):
    """Scores that reach far apart, values whose scales do, in every order; heads of queries that are zero."""
    n = [200, 64, 1000]
    pool, scale = _cache(90, 2, 128, kind)
    ptr, idx, last = _lists(n, 90, 3)
    scale[:, 0] *= torch.exp(2 * torch.randn(90, 2, 16, device="cuda"))
    scale[int(idx[2]), 1, :, 7] *= 2.0 ** 8                       # one value far larger than the others, in the middle
    q = torch.randn(3, 16 * 128, device="cuda").to(torch.bfloat16) * 6
    q[1, :128] = 0
    q[2] *= 2.0 ** -20
    args = (pool, scale, torch.arange(4, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=3, q_heads=16, kv_heads=2, head_dim=128, prefix_len=500)
    out = torch.empty_like(q)
    ops.attn_decode_q8(q, out, *args, q_heads=16, req_begin=0, req_count=3, workspace=ws)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=16, req_begin=0, req_count=3), 128)
    front = idx[:32].contiguous()
    ops.attn_decode_shared_q8(q, out, *args, front, 500, q_heads=16, req_begin=0, req_count=3, workspace=ws)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=16, req_begin=0, req_count=3, prefix_pages=front, prefix_len=500), 128)


@KINDS
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (7, 1, 128), (16, 1, 64), (9, 3, 64)])
@pytest.mark.parametrize("requests,prefix,own", [(1, 1, [1]), (5, 15, [0, 1, 2, 0, 16]), (40, 64, [i % 37 for i in range(40)]), (3, 65, [0, 0, 0]),
                                                 (16, 1999, [3 * i for i in range(16)]), (130, 700, [i % 50 for i in range(130)]),
                                                 (2, 9000, [5000, 1])])
def test_shared_prefix(kind, heads, kv_heads, dim, requests, prefix, own):
    pages = sum(-(-x // 16) for x in own) + -(-prefix // 16) + 2
    pool, scale = _cache(pages, kv_heads, dim, kind)
    order = random.Random(8).sample(range(pages), pages)
    front, rest = order[:-(-prefix // 16)], order[-(-prefix // 16):]
    ptr, idx, last = _lists(own, len(rest), 5)
    idx = _i32([rest[i] for i in idx.tolist()])
    q = torch.randn(requests + 1, heads * dim, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 3.0)
    args = (pool, scale, torch.arange(requests + 1, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=requests, q_heads=heads, kv_heads=kv_heads, head_dim=dim, prefix_len=prefix)
    st = ops.new_status()
    ops.attn_decode_shared_q8(q, out, *args, _i32(front), prefix, q_heads=heads, req_begin=0, req_count=requests, workspace=ws, status=st)
    ops.check_status(st)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=heads, req_begin=0, req_count=requests, prefix_pages=_i32(front), prefix_len=prefix), dim)
    assert bool((out[requests:] == 3).all())
    same = torch.empty_like(out)
    ops.attn_decode_shared_q8(q, same, *args, _i32(front), prefix, q_heads=heads, req_begin=0, req_count=requests, workspace=ws)
    assert torch.equal(same[:requests], out[:requests])


@pytest.mark.parametrize("prefix", [0, 100])
def test_more_requests_than_a_block_lists(prefix):
    own = [(37 * i) % 23 for i in range(1100)]
    pages = sum(-(-x // 16) for x in own) + 7
    pool, scale = _cache(pages, 2, 64, INT8)
    ptr, idx, last = _lists(own, pages - 7, 5)
    front = torch.arange(pages - 7, pages, dtype=torch.int32, device="cuda")
    q = torch.randn(1100, 2 * 64, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    args = (pool, scale, torch.arange(1101, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=1100, q_heads=2, kv_heads=2, head_dim=64, prefix_len=prefix)
    ops.attn_decode_shared_q8(q, out, *args, front, prefix, q_heads=2, req_begin=0, req_count=1100, workspace=ws)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=2, req_begin=0, req_count=1100, prefix_pages=front, prefix_len=prefix), 64)


@pytest.mark.parametrize("heads,kv_heads,requests,prefix,ctas", [(8, 2, 5, 5000, 3), (16, 4, 70, 3333, 7), (16, 4, 70, 3333, 0), (3, 1, 2, 9001, 40), (32, 8, 9, 700, 5)])
def test_shared_prefix_over_few_ctas(heads, kv_heads, requests, prefix, ctas):
    """Shares with the ends of several items, shares that end where an item begins."""
    pages = -(-prefix // 16)
    pool, scale = _cache(pages + 60, kv_heads, 64, E4M3, seed=4)
    ptr, idx, last = _lists([(7 * i) % 12 for i in range(requests)], pages + 60, 6)
    front = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).contiguous()
    q = torch.randn(requests, heads * 64, device="cuda").to(torch.bfloat16)
    args = (pool, scale, torch.arange(requests + 1, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=requests, q_heads=heads, kv_heads=kv_heads, head_dim=64, prefix_len=prefix)
    ws.fill_(255)
    out, st = torch.zeros_like(q), ops.new_status()
    ops.attn_decode_shared_q8(q, out, *args, front, prefix, q_heads=heads, req_begin=0, req_count=requests, workspace=ws, num_ctas=ctas, status=st)
    ops.check_status(st)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=heads, req_begin=0, req_count=requests, prefix_pages=front, prefix_len=prefix), 64)


def test_no_prefix_is_plain_decode():
    pool, scale = _cache(40, 2, 128, E4M3)
    ptr, idx, last = _lists([100, 7, 333], 40, 3)
    q = torch.randn(3, 8 * 128, device="cuda").to(torch.bfloat16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    args = (pool, scale, torch.arange(4, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=3, q_heads=8, kv_heads=2, head_dim=128)
    ops.attn_decode_q8(q, a, *args, q_heads=8, req_begin=0, req_count=3, workspace=ws)
    ops.attn_decode_shared_q8(q, b, *args, None, 0, q_heads=8, req_begin=0, req_count=3, workspace=ws)
    assert torch.equal(a, b)


@pytest.mark.parametrize("prefix,lengths", [(0, [3]), (0, [900, 0, 35, 1]), (0, [4000] * 5 + [17]), (130, [40, 0, 200]), (9000, [0])])
def test_workspace_may_hold_anything(prefix, lengths):
    """NaN and large words in the workspace, and one made for more requests and a longer prefix: the same rows."""
    pool, scale = _cache(2000, 2, 128, E4M3)
    ptr, idx, last = _lists(lengths, 2000, 3)
    n = len(lengths)
    q = torch.randn(n, 8 * 128, device="cuda").to(torch.bfloat16)
    front = torch.arange(-(-prefix // 16), dtype=torch.int32, device="cuda")
    sizes = dict(q_heads=8, kv_heads=2, head_dim=128)
    made = [ops.decode_workspace_q8(requests=r, prefix_len=p, **sizes) for r, p in ((n, prefix), (n, prefix), (n + 60, prefix + 70))]
    outs = []
    for ws, byte in zip(made, (0, 255, 127)):
        ws.fill_(byte)
        outs.append(ops.attn_decode_shared_q8(q, torch.empty_like(q), pool, scale, torch.arange(n + 1, dtype=torch.int32, device="cuda"), ptr, idx,
                                              last, front, prefix, q_heads=8, req_begin=0, req_count=n, workspace=ws))
    assert bool(outs[0].isfinite().all()) and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("lengths", [([30, 5], [17, 18]), ([900, 33, 250, 1000], [3, 1500, 1, 600])])
def test_kernels_that_start_early_see_what_the_ones_before_wrote(lengths):
    """Lists, queries and the cache change in front of every call, on one stream without a wait: the rows of calls one by one."""
    heads, kv_heads, dim, n = 8, 2, 128, len(lengths[0])
    pool, scale = _cache(300, kv_heads, dim, E4M3)
    keep = pool.clone(), scale.clone()
    sets = [_lists(x, 250, 5 + i) for i, x in enumerate(lengths)]
    size = max(idx.numel() for _, idx, _ in sets)
    sets = [(ptr, torch.nn.functional.pad(idx, (0, size - idx.numel())), last) for ptr, idx, last in sets]
    qkv = [torch.randn(n, (heads + 2 * kv_heads) * dim, device="cuda").to(torch.bfloat16) for _ in sets]
    lists, row, q = [torch.empty_like(t) for t in sets[0]], torch.empty_like(qkv[0]), torch.empty(n, heads * dim, dtype=torch.bfloat16, device="cuda")
    front, qo = torch.arange(250, 290, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    ws = ops.decode_workspace_q8(requests=n, q_heads=heads, kv_heads=kv_heads, head_dim=dim, prefix_len=630)
    freq = torch.rand(dim // 2, device="cuda")

    def run(early, wait):
        pool.view(torch.uint8).copy_(keep[0].view(torch.uint8))
        scale.copy_(keep[1])
        outs = []
        for i in range(12):
            for to, new in zip(lists, sets[i & 1]):
                to.copy_(new)
            row.copy_(qkv[i & 1])
            position = (lists[0][1:] - lists[0][:-1]) * 16 - 16 + lists[2] - 1
            ops.rope_append_q8(row, q, pool, scale, freq, position.int(), qo[:n], lists[0], lists[1], q_heads=heads, kv_heads=kv_heads, head_dim=dim,
                               q_off=0, k_off=heads * dim, v_off=(heads + kv_heads) * dim, early_start=early & 1)
            a = ops.attn_decode_q8(q, torch.zeros_like(q), pool, scale, qo, *lists, q_heads=heads, req_begin=0, req_count=n, workspace=ws,
                                   early_start=early)
            b = ops.attn_decode_shared_q8(q, torch.zeros_like(q), pool, scale, qo, *lists, front, 630, q_heads=heads, req_begin=0, req_count=n,
                                          workspace=ws, early_start=early)
            outs += [a, b, ops.kv_read_q8(pool, scale, lists[1], early_start=early & 1)]
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    want = run(0, True)
    for early in (0, 1, 2, 3, 3):
        assert all(torch.equal(x, y) for x, y in zip(run(early, False), want))


def test_lists_that_are_none_are_reported():
    """Page numbers, rows and page lists out of range: a status, finite rows, and a workspace that still serves."""
    pool, scale = _cache(40, 2, 128, E4M3)
    ptr, idx, last = _lists([100, 7, 333], 40, 3)
    q = torch.randn(3, 8 * 128, device="cuda").to(torch.bfloat16)
    out = torch.zeros_like(q)
    qo = torch.arange(4, dtype=torch.int32, device="cuda")
    ws = ops.decode_workspace_q8(requests=3, q_heads=8, kv_heads=2, head_dim=128, prefix_len=40)
    st = ops.new_status()

    def wrong(qo=qo, ptr=ptr, idx=idx, front=None):
        kw = dict(q_heads=8, req_begin=0, req_count=3, workspace=ws, status=st)
        if front is None:
            ops.attn_decode_q8(q, out, pool, scale, qo, ptr, idx, last, **kw)
        else:
            ops.attn_decode_shared_q8(q, out, pool, scale, qo, ptr, idx, last, front, 40, **kw)
        with pytest.raises(RuntimeError, match="out-of-range"):
            ops.check_status(st)
        assert bool(out.isfinite().all())

    wrong(idx=torch.where(idx == idx[3], -5, idx))
    wrong(idx=torch.where(idx == idx[3], 40, idx))
    wrong(qo=_i32([0, 3, 1, 2]))
    wrong(qo=_i32([0, -1, 1, 2]))
    wrong(ptr=_i32([0, 9, 8, 29]))
    wrong(ptr=_i32([0, 7, 8, 60]))
    wrong(ptr=_i32([-3, 7, 8, 29]))
    wrong(front=_i32([1, 2, 77]))
    args = (pool, scale, qo, ptr, idx, last)
    ops.attn_decode_q8(q, out, *args, q_heads=8, req_begin=0, req_count=3, workspace=ws, status=st)
    ops.check_status(st)
    _check_rows(out, ref.attn_decode_q8(q, *args, q_heads=8, req_begin=0, req_count=3), 128)


def test_offsets_beyond_32_bits():
    """A pool of over 4 GB whose last pages are the ones that are written and read."""
    kv_heads, dim, pages = 8, 128, 140000
    pool, scale = ops.kv_pool_q8(pages, kv_heads, dim, torch.int8)
    small, small_scale = _cache(8, kv_heads, dim, INT8)
    pool[-8:], scale[-8:] = small, small_scale
    ids = _i32(range(pages - 8, pages))
    assert torch.equal(ops.kv_read_q8(pool, scale, ids), ops.kv_read_q8(small, small_scale, _i32(range(8))))
    q = torch.randn(2, 32 * dim, device="cuda").to(torch.bfloat16)
    ws = ops.decode_workspace_q8(requests=2, q_heads=32, kv_heads=kv_heads, head_dim=dim, prefix_len=50)
    outs = []
    for p, s, first in ((pool, scale, pages - 8), (small, small_scale, 0)):
        idx, out = _i32([first + 5, first + 6, first + 7]), torch.empty_like(q)
        ops.attn_decode_shared_q8(q, out, p, s, _i32([0, 1, 2]), _i32([0, 2, 3]), idx, _i32([3, 9]), _i32(range(first, first + 4)), 50, q_heads=32,
                                  req_begin=0, req_count=2, workspace=ws)
        outs.append(out)
    assert torch.equal(*outs)
    qkv = torch.randn(1, 48 * dim, device="cuda").to(torch.bfloat16)
    row = torch.empty(1, 32 * dim, dtype=torch.bfloat16, device="cuda")
    for p, s, first in ((pool, scale, pages - 8), (small, small_scale, 0)):
        ops.rope_append_q8(qkv, row, p, s, torch.ones(64, device="cuda"), _i32([20]), _i32([0]), _i32([0, 2]), _i32([first, first + 7]), q_heads=32,
                           kv_heads=kv_heads, head_dim=dim, q_off=16 * dim, k_off=0, v_off=8 * dim)
    assert torch.equal(pool[-1], small[-1]) and torch.equal(scale[-1], small_scale[-1])


# ---- streams, graphs, and a run of them together -------------------------------------------------------------------------
def test_two_streams_and_a_captured_graph():
    pool, scale = _cache(200, 2, 128, E4M3)
    ptr, idx, last = _lists([1500, 7, 333, 40], 150, 3)
    front = _i32(sorted(set(range(200)) - set(idx.tolist()))[:40])
    q = torch.randn(4, 8 * 128, device="cuda").to(torch.bfloat16)
    qo = torch.arange(5, dtype=torch.int32, device="cuda")
    args = (pool, scale, qo, ptr, idx, last)
    kw = dict(q_heads=8, req_begin=0, req_count=4)
    make = lambda: ops.decode_workspace_q8(requests=4, q_heads=8, kv_heads=2, head_dim=128, prefix_len=600)
    want, want_s = torch.empty_like(q), torch.empty_like(q)
    ws = make()
    ops.attn_decode_q8(q, want, *args, **kw, workspace=ws)
    ops.attn_decode_shared_q8(q, want_s, *args, front, 600, **kw, workspace=ws)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [(torch.empty_like(q), torch.empty_like(q), make()) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (a, b, w) in zip(streams, outs):
            with torch.cuda.stream(s):
                ops.attn_decode_q8(q, a, *args, **kw, workspace=w)
                ops.attn_decode_shared_q8(q, b, *args, front, 600, **kw, workspace=w)
    torch.cuda.synchronize()
    for a, b, _ in outs:
        assert torch.equal(a, want) and torch.equal(b, want_s)
    # captured once, replayed with other lengths in the same buffers
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_decode_shared_q8(q, out, *args, front, 600, **kw, workspace=ws)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_s)
    ptr.copy_(_i32([0, 20, 20, 90, 119]))
    last.copy_(_i32([16, 0, 2, 9]))
    q.copy_(torch.randn(4, 8 * 128))
    graph.replay()
    torch.cuda.synchronize()
    _check_rows(out, ref.attn_decode_q8(q, *args, **kw, prefix_pages=front, prefix_len=600), 128)


@KINDS
def test_prompt_and_decode_steps_on_one_cache(kind):
    """A shared system prompt, two requests behind it: the prompts' tokens are cached and attended with the prefill kernel on pages
    that are read back, then single tokens follow, all against attention in 64 bits over what the cache holds."""
    heads, kv_heads, dim = 8, 2, 128
    width = (heads + 2 * kv_heads) * dim
    cols = dict(q_heads=heads, kv_heads=kv_heads, head_dim=dim, q_off=2 * kv_heads * dim, k_off=0, v_off=kv_heads * dim)
    pool, scale = ops.kv_pool_q8(64, kv_heads, dim, kind)
    inv = (10000.0 ** (-torch.arange(0, dim, 2, device="cuda").double() / dim)).float()
    norms = dict(q_norm=torch.ones(dim, dtype=torch.bfloat16, device="cuda"), k_norm=torch.ones(dim, dtype=torch.bfloat16, device="cuda"))
    st = ops.new_status()

    def append(n, req, positions, ptr, idx):
        qkv, q = torch.randn(n, width, device="cuda").to(torch.bfloat16), torch.empty(n, heads * dim, dtype=torch.bfloat16, device="cuda")
        ops.rope_append_q8(qkv, q, pool, scale, inv, _i32(positions), _i32(req), ptr, idx, **cols, **norms, status=st)
        return q

    # the system prompt: 90 tokens, pages 3, 60, 7, 8, 40, 2
    front = _i32([3, 60, 7, 8, 40, 2])
    q = append(90, [0] * 90, range(90), _i32([0, 6]), front)
    pages = ops.kv_read_q8(pool, scale, front, status=st)
    out = torch.empty_like(q)
    items = _i32([[0, t, min(32, 90 - t)] for t in range(0, 90, 32)])
    ops.attn_prefill(q, out, pages, _i32([0, 90]), _i32([0, 6]), torch.arange(6, dtype=torch.int32, device="cuda"), _i32([10]), items,
                     q_heads=heads, status=st)
    ops.check_status(st)
    values = ref.kv_values_q8(pool, scale, front).permute(1, 2, 0, 3, 4).reshape(2, kv_heads, 96, dim)[:, :, :90]
    s = torch.einsum("tgrd,gjd->grtj", q.double().cpu().view(90, kv_heads, heads // kv_heads, dim), values[0]) * dim ** -0.5
    p = torch.softmax(s.masked_fill(torch.ones(90, 90).triu(1).bool(), -torch.inf), -1)
    want, size = (torch.einsum("grtj,gjd->tgrd", p, x).reshape(90, -1) for x in (values[1], values[1].abs()))
    # the pages as bf16 (2^-8 of keys and values; a score is a sum of up to 128 products of normal numbers, its error below 0.03),
    # weights in bf16
    assert bool(((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + size * (2 * 2.0 ** -8 + 0.06)).all())
    # two requests behind it (their positions go on from the 90 tokens; their own pages hold what follows the prompt)
    own = _i32([10, 11, 12, 20, 21])
    ptr = _i32([0, 3, 5])
    lengths = [0, 0]
    ws = ops.decode_workspace_q8(requests=2, q_heads=heads, kv_heads=kv_heads, head_dim=dim, prefix_len=90)
    for step in range(20):
        # slots count from the request's own first page, so that its tokens' positions in the list are what is passed
        q = append(2, [0, 1], lengths, ptr, own)
        lengths = [n + 1 for n in lengths]
        counts = [-(-n // 16) for n in lengths]
        lists = (_i32([0, 1, 2]), _i32([0, counts[0], sum(counts)]), _i32(own[:counts[0]].tolist() + own[3:3 + counts[1]].tolist()),
                 _i32([n - 16 * (c - 1) for n, c in zip(lengths, counts)]))
        out = torch.empty_like(q)
        ops.attn_decode_shared_q8(q, out, pool, scale, *lists, front, 90, q_heads=heads, req_begin=0, req_count=2, workspace=ws, status=st)
        ops.check_status(st)
        _check_rows(out, ref.attn_decode_q8(q, pool, scale, *lists, q_heads=heads, req_begin=0, req_count=2, prefix_pages=front, prefix_len=90), dim)
        if step % 7 == 0:                         # the same over one list of pages, where the prompt fills whole ones: another cut, other sums
            whole = _i32(front[:5].tolist() + own[:counts[0]].tolist())
            one = torch.empty_like(q)
            ops.attn_decode_q8(q, one, pool, scale, _i32([0, 1]), _i32([0, len(whole)]), whole, lists[3][:1].contiguous(), q_heads=heads, req_begin=0,
                               req_count=1, workspace=ws, status=st)
            two = torch.empty_like(q)
            ops.attn_decode_shared_q8(q, two, pool, scale, *lists, front, 80, q_heads=heads, req_begin=0, req_count=1, workspace=ws, status=st)
            ops.check_status(st)
            assert bool(((one[0] - two[0]).abs().float() <= 0.02 * one[0].abs().float() + 0.01 * one[0].abs().max()).all())


def _refusal_arguments():
    pool, scale = _cache(6, 2, 64, INT8)
    ptr, idx, last = _lists([20, 30], 6, 1, extra=1)
    x = torch.randn(2, 8 * 64, device="cuda").to(torch.bfloat16)
    append = dict(qkv=x, q_out=torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device="cuda"), kv_pool=pool, kv_scale=scale,
                  inv_freq=torch.ones(32, device="cuda"), positions=_i32([3, 4]), token_req=_i32([0, 1]), kv_indptr=ptr, kv_indices=idx, q_heads=4,
                  kv_heads=2, head_dim=64, q_off=0, k_off=256, v_off=384, status=None)
    read = dict(kv_pool=pool, kv_scale=scale, page_ids=_i32([1, 2]), out=torch.zeros(2, 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda"))
    q = x[:, :256].contiguous()
    decode = dict(q=q, out=torch.zeros_like(q), kv_pool=pool, kv_scale=scale, qo_indptr=_i32([0, 1]), kv_indptr=ptr, kv_indices=idx,
                  kv_last_page_len=last, prefix_pages=_i32([0, 1]), prefix_len=20, q_heads=4, req_begin=0, req_count=2,
                  workspace=ops.decode_workspace_q8(requests=2, q_heads=4, kv_heads=2, head_dim=64, prefix_len=20))
    return {"append": (ops.rope_append_q8, append, "q_out"), "read": (ops.kv_read_q8, read, "out"), "decode": (ops.attn_decode_shared_q8, decode, "out")}


@pytest.mark.parametrize("op,change,why", [
    ("append", lambda a: dict(qkv=a["qkv"].float()), "bfloat16"), ("append", lambda a: dict(qkv=a["qkv"].t()), "unit inner stride"),
    ("append", lambda a: dict(qkv=a["qkv"].cpu()), "on cuda"), ("append", lambda a: dict(q_out=a["q_out"][:1]), "q_out"),
    ("append", lambda a: dict(q_out=a["qkv"][:, :256].contiguous().t().contiguous().t()), "q_out"),
    ("append", lambda a: dict(q_out=a["qkv"].view(-1)[256:768].view(2, 256)), "overlap"),
    ("append", lambda a: dict(k_off=-8), "columns"), ("append", lambda a: dict(v_off=392), "columns"), ("append", lambda a: dict(k_off=260), "alignment"),
    ("append", lambda a: dict(q_heads=2 ** 31), "32 bits"), ("append", lambda a: dict(kv_heads=4), "these heads"),
    ("append", lambda a: dict(head_dim=128), "these heads"), ("append", lambda a: dict(kv_scale=a["kv_scale"].view(-1)), "kv_scale"),
    ("append", lambda a: dict(kv_pool=a["kv_pool"].view(torch.uint8)), "kv_pool"), ("append", lambda a: dict(positions=a["positions"].long()), "int32"),
    ("append", lambda a: dict(token_req=a["token_req"][:1]), "per token"), ("append", lambda a: dict(kv_indptr=a["kv_indptr"][:1]), "per request"),
    ("append", lambda a: dict(inv_freq=a["inv_freq"][:16]), "inv_freq"), ("append", lambda a: dict(q_norm=torch.ones(32, dtype=torch.bfloat16, device="cuda")), "norms"),
    ("append", lambda a: dict(k_norm=torch.ones(64, device="cuda")), "bfloat16"), ("append", lambda a: dict(cos_sin=a["inv_freq"]), "cos_sin"),
    ("append", lambda a: dict(eps="small"), "number"), ("append", lambda a: dict(status=a["positions"][:0]), "status"),
    ("read", lambda a: dict(out=a["out"][:1]), "pages"), ("read", lambda a: dict(out=a["out"].half()), "bfloat16"),
    ("read", lambda a: dict(page_ids=a["page_ids"].long()), "int32"), ("read", lambda a: dict(page_ids=[1, 2]), "tensor"),
    ("read", lambda a: dict(kv_pool=a["kv_pool"][:, :, :, :, :32]), "kv_pool"), ("read", lambda a: dict(kv_scale=a["kv_scale"][:3]), "kv_scale"),
    ("read", lambda a: dict(out=a["kv_pool"].view(-1).view(torch.bfloat16)[:4096].view(1, 2, 2, 16, 64), page_ids=a["page_ids"][:1]), "overlap"),
    ("decode", lambda a: dict(q_heads=3), "KV head"), ("decode", lambda a: dict(q_heads=34), "KV head"), ("decode", lambda a: dict(q_heads=0), "KV head"),
    ("decode", lambda a: dict(q_heads=2), "q and out"), ("decode", lambda a: dict(out=a["out"][:1]), "q and out"), ("decode", lambda a: dict(out=a["q"]), "overlap"),
    ("decode", lambda a: dict(q=a["q"].half()), "bfloat16"), ("decode", lambda a: dict(req_count=3), "listed"), ("decode", lambda a: dict(req_begin=1), "listed"),
    ("decode", lambda a: dict(req_begin=-1), "listed"), ("decode", lambda a: dict(kv_last_page_len=a["kv_last_page_len"][:1]), "listed"),
    ("decode", lambda a: dict(prefix_len=-1), "negative"), ("decode", lambda a: dict(prefix_len=33), "prefix_pages"),
    ("decode", lambda a: dict(prefix_pages=None), "prefix_pages"), ("decode", lambda a: dict(workspace=None), "workspace"),
    ("decode", lambda a: dict(workspace=a["workspace"][256:]), "bad argument"), ("decode", lambda a: dict(workspace=a["workspace"][1:]), "bad argument"),
    ("decode", lambda a: dict(num_ctas=-1), "bad argument"), ("decode", lambda a: dict(sm_scale="small"), "number"),
    ("decode", lambda a: dict(kv_indices=a["kv_indices"].cpu()), "on cuda")])
def test_calls_refuse(op, change, why):
    """Arguments that do not fit are refused by the host, and nothing is written."""
    call, args, written = _refusal_arguments()[op]
    before = [args[k].clone() for k in (written, "kv_scale")]
    with pytest.raises(RuntimeError, match=why):
        call(**{**args, **change(args)})
    torch.cuda.synchronize()
    assert all(torch.equal(args[k], b) for k, b in zip((written, "kv_scale"), before))


def test_the_calls_behind_the_refusals_serve():
    for call, args, written in _refusal_arguments().values():
        call(**args)
        assert bool(args[written].any()) and bool(args[written].isfinite().all())
