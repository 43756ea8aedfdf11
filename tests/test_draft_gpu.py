"""Drafted tokens on the GPU: each operator against its plain form in 64 bits, the edges of its range, and a run of all of them.

Tolerances. Outputs are rounded to bf16 once: 2^-8 of the value. Attention's weights are rounded to bf16 before the product, 2^-8 of each, so
that a row is off by up to 2^-8 of sum p |v| more; scores are fp32 sums of up to 128 products (2^-24 128 sum |q k| scale, below 2^-11 for
normal queries and keys), which the weights carry on: 2^-10 of sum p |v| covers these and 2^x."""
import math
import random

import pytest
import torch

from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

PAGE = 16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0):
    return torch.empty(*shape, device="cuda").normal_(0, std, generator=g).to(torch.bfloat16)


# ---- tables -----------------------------------------------------------------------------------------------------------
def _tables(rows, max_pages, num_pages, lengths, seed=0):
    """Tables with requests of the given lengths, in pages dealt out at random, and a CPU copy."""
    g = torch.Generator().manual_seed(seed)
    t = ops.page_tables(rows, max_pages, num_pages, "cpu")
    t.free_pages.copy_(torch.randperm(num_pages, generator=g))
    t.table.copy_(torch.randint(0, num_pages, t.table.shape, generator=g))         # what lies behind a row's pages does not matter
    ref.tables_grow(t.table, t.lengths, t.free_pages, t.free_count, torch.arange(rows), torch.tensor(lengths))
    return ops.PageTables(*(x.cuda() for x in (t.table, t.lengths, t.free_pages, t.free_count))), t


def _same_tables(t, c):
    for f in ("table", "lengths", "free_pages", "free_count"):
        assert torch.equal(getattr(t, f).cpu(), getattr(c, f)), f
    assert t.ticket.item() == 0


def _same_lists(li, want, R, last=0, kept=None):
    n, pages = len(want["slots"]), len(want["kv_indices"])
    for f in ("qo_indptr", "kv_indptr"):
        assert getattr(li, f)[:R + 1].tolist() == want[f], f
    assert li.kv_last_page_len[:R].tolist() == want["kv_last_page_len"]
    assert li.kv_indices[:pages].tolist() == want["kv_indices"]
    if kept is not None:
        assert torch.equal(li.kv_indices[pages:], kept[pages:])
    for f, rest in (("positions", 0), ("token_req", -1), ("slots", -1)):
        assert getattr(li, f).tolist() == want[f] + [rest] * (getattr(li, f).numel() - n), f


@pytest.mark.parametrize("R,lo,hi,new,spare", [(1, 0, 0, 1, 0), (1, 15, 15, 1, 3), (1, 16, 16, 1, 0), (1, 2000, 2000, 600, 5), (7, 0, 50, 40, 100), (33, 0, 400, 3, 1),
                                               (513, 0, 200, 9, 0), (1000, 1, 30, 20, 7), (4096, 0, 60, 2, 0), (3, 20000, 40000, 2000, 64)])
def test_grow_and_trim(R, lo, hi, new, spare):
    r = random.Random(R * 1000 + hi)
    rows = R + r.randint(0, 5)
    lengths = [r.randint(lo, hi) for _ in range(rows)]
    most = (hi + 2 * new) // PAGE + 2
    t, c = _tables(rows, most, rows * most, lengths)
    order = r.sample(range(rows), R)
    for step in range(2):
        n = [r.choice([0, 1, new, r.randint(0, new)]) for _ in range(R)]
        want = ref.tables_grow(c.table, c.lengths, c.free_pages, c.free_count, torch.tensor(order), torch.tensor(n))
        li = ops.batch_lists(R, sum(n) + spare, len(want["kv_indices"]) + spare)
        li.kv_indices.random_(0, 1000)
        kept = li.kv_indices.clone()
        status = ops.new_status()
        assert ops.tables_grow(t, i32(order), i32(n), li, status=status) is li
        ops.check_status(status)
        _same_lists(li, want, R, kept=kept)
        _same_tables(t, c)
        drop = [r.choice([0, 1, k, r.randint(0, k)]) for k in n] if step == 0 else [r.choice([0, 10 ** 9, r.randint(0, hi + 1)]) for _ in n]
        ops.tables_trim(t, i32(order), i32(drop), status=status)
        ref.tables_trim(c.table, c.lengths, c.free_pages, c.free_count, torch.tensor(order), torch.tensor(drop))
        ops.check_status(status)
        _same_tables(t, c)


def test_trim_takes_back_a_grow():
    t, c = _tables(6, 20, 90, [0, 5, 16, 100, 31, 64])
    n = i32([40, 1, 16, 0, 3, 33])
    ops.tables_grow(t, i32([3, 1, 0, 2, 5, 4]), n, ops.batch_lists(6, 100, 90))
    ops.tables_trim(t, i32([3, 1, 0, 2, 5, 4]), n)
    for f in ("lengths", "free_pages", "free_count"):
        assert torch.equal(getattr(t, f).cpu(), getattr(c, f))


@pytest.mark.parametrize("rows,new,change", [
    ([0, 6], [1, 1], {}), ([0, -1], [1, 1], {}), ([2, 2], [1, 1], {}), ([1, 3], [1, -1], {}), ([1, 3], [200, 1], {}), ([1, 3], [2 ** 31 - 1, 2 ** 31 - 1], {}),
    ([1, 3], [5, 5], {"free_count": 0}), ([1, 3], [5, 5], {"free_count": -1}), ([1, 3], [5, 5], {"free_count": 91}), ([1, 3], [5, 5], {"tokens": 9}),
    ([1, 3], [5, 5], {"pages": 5}), ([1, 3], [5, 5], {"length": -1}), ([1, 3], [5, 5], {"length": 321})])
def test_grow_that_does_not_fit_changes_nothing(rows, new, change):
    t, _ = _tables(6, 20, 90, [0, 15, 16, 100, 31, 64])
    if "free_count" in change:
        t.free_count.fill_(change["free_count"])
    if "length" in change:
        t.lengths[3] = change["length"]
    before = [x.clone() for x in (t.table, t.lengths, t.free_pages, t.free_count)]
    li = ops.batch_lists(2, change.get("tokens", 40), change.get("pages", 40))
    for x in (li.qo_indptr, li.kv_indptr, li.kv_last_page_len, li.slots, li.positions):
        x.fill_(7)
    status = ops.new_status()
    ops.tables_grow(t, i32(rows), i32(new), li, status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    for a, b in zip(before, (t.table, t.lengths, t.free_pages, t.free_count)):
        assert torch.equal(a, b)
    assert not any(x.any() for x in (li.qo_indptr, li.kv_indptr, li.kv_last_page_len, li.positions)) and (li.slots == -1).all() and (li.token_req == -1).all()
    if not change.get("tokens") and not change.get("pages") and new[0] < 200 and change.get("free_count") != 0:
        ops.tables_trim(t, i32(rows), i32(new), status=status)
        with pytest.raises(RuntimeError, match="index"):
            ops.check_status(status)
        for a, b in zip(before, (t.table, t.lengths, t.free_pages, t.free_count)):
            assert torch.equal(a, b)


def test_trim_beyond_the_pool_changes_nothing():
    t, _ = _tables(6, 20, 90, [0, 15, 16, 100, 31, 64])
    t.free_count.fill_(85)
    before = t.lengths.clone()
    status = ops.new_status()
    ops.tables_trim(t, i32([3]), i32([100]), status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert torch.equal(before, t.lengths) and t.free_count.item() == 85


def test_tables_of_empty_batches():
    t, c = _tables(3, 4, 12, [5, 0, 33])
    li = ops.batch_lists(0, 3, 2)
    ops.tables_grow(t, i32([]), i32([]), li)
    assert li.qo_indptr.tolist() == [0] and li.slots.tolist() == [-1] * 3
    li = ops.batch_lists(1, 0, 5)
    ops.tables_grow(t, i32([2]), i32([0]), li)
    assert li.kv_indptr.tolist() == [0, 3] and li.kv_last_page_len.tolist() == [1]
    ops.tables_trim(t, i32([]), i32([]))
    _same_tables(t, c)


# ---- rotation -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,G,d,pairs,interleaved,factor,far", [
    (1, 1, 1, 64, 32, False, 1.0, 10), (5, 32, 8, 128, 64, False, 1.0, 1000000), (9, 9, 3, 64, 32, True, 1.0, 5000), (17, 28, 4, 128, 32, False, 1.25, 100000),
    (17, 28, 4, 128, 32, True, 1.25, 100000), (33, 5, 5, 128, 10, False, 1.0, 3000), (33, 5, 5, 128, 10, True, 1.0, 3000), (4, 2, 1, 64, 1, False, 0.5, 77),
    (4, 2, 1, 64, 1, True, 0.5, 77), (300, 16, 1, 128, 48, False, 1.0, 2 ** 31 - 1), (7, 3, 3, 64, 24, False, 1.0, 40), (7, 3, 3, 64, 31, False, 1.0, 40)])
def test_rotation(T, H, G, d, pairs, interleaved, factor, far):
    g = gen(T + d + pairs)
    pages = T // PAGE + 3
    # columns: values, some that nobody reads, queries, keys; rows further apart than their length
    v_off, q_off, k_off = 0, G * d + 8, G * d + 8 + H * d
    wide = normal(g, T, (H + 2 * G) * d + 24, std=3.0)
    qkv = wide[:, :(H + 2 * G) * d + 8]
    inv = (10000.0 ** (-torch.arange(pairs, device="cuda").double() / pairs)).float()
    pos = torch.randint(0, far, (T,), generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(pages * PAGE, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1                                    # padding
    pool = normal(g, pages, 2, G, PAGE, d)
    before, q = pool.clone(), torch.full((T, H * d), 7.0, dtype=torch.bfloat16, device="cuda")
    status = ops.new_status()
    ops.rope_append_slots(qkv, q, pool, inv, pos, slots, q_heads=H, kv_heads=G, head_dim=d, q_off=q_off, k_off=k_off, v_off=v_off, interleaved=interleaved,
                          factor=factor, status=status)
    ops.check_status(status)
    x = qkv.double()
    want_q = ref.rope_layout(x[:, q_off:q_off + H * d].view(T, H, d), pos, inv, interleaved, factor)
    want_k = ref.rope_layout(x[:, k_off:k_off + G * d].view(T, G, d), pos, inv, interleaved, factor)
    size = x.abs().max().item() * max(1.0, factor) * 2   # |x cos| + |y sin|; the angle is good to 2^-22, an fp32 sum of two to 2^-23

    def near(got, want):
        assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -21).all()

    near(q.view(T, H, d), want_q)
    rest = slice(2 * pairs, d)
    assert torch.equal(q.view(T, H, d)[..., rest], qkv[:, q_off:q_off + H * d].reshape(T, H, d)[..., rest])
    for t in range(T):
        s = int(slots[t])
        if s < 0:
            continue
        near(pool[s // PAGE, 0, :, s % PAGE], want_k[t])
        assert torch.equal(pool[s // PAGE, 1, :, s % PAGE], qkv[t, v_off:v_off + G * d].view(G, d))
        before[s // PAGE, :, :, s % PAGE] = pool[s // PAGE, :, :, s % PAGE]
    assert torch.equal(before, pool)                     # nothing else


def test_rotation_of_what_is_not_finite_stays_in_its_pair():
    d, inf = 64, float("inf")
    qkv = normal(gen(1), 2, 3 * d)
    qkv[0, 5], qkv[0, d + 40], qkv[0, 2 * d + 3], qkv[1, 50] = inf, float("nan"), -inf, inf
    pool, q = torch.zeros(1, 2, 1, PAGE, d, dtype=torch.bfloat16, device="cuda"), torch.empty(2, d, dtype=torch.bfloat16, device="cuda")
    inv = torch.full((16,), 0.3, device="cuda")
    ops.rope_append_slots(qkv, q, pool, inv, i32([3, 4]), i32([2, 9]), q_heads=1, kv_heads=1, head_dim=d, q_off=0, k_off=d, v_off=2 * d)
    assert (~q[0].isfinite()).nonzero().flatten().tolist() == [5, 21]
    assert (~q[1].isfinite()).nonzero().flatten().tolist() == [50] and q[1, 50] == inf
    assert (~pool[0, 0, 0, 2].isfinite()).nonzero().flatten().tolist() == [40]
    assert (~pool[0, 1, 0, 2].isfinite()).nonzero().flatten().tolist() == [3]


def test_rotation_reports_slots_that_do_not_exist():
    d = 64
    qkv, pool = normal(gen(1), 3, 3 * d), torch.zeros(2, 2, 1, PAGE, d, dtype=torch.bfloat16, device="cuda")
    q, status = torch.empty(3, d, dtype=torch.bfloat16, device="cuda"), ops.new_status()
    ops.rope_append_slots(qkv, q, pool, torch.ones(32, device="cuda"), i32([0, 0, 0]), i32([32, 31, -5]), q_heads=1, kv_heads=1, head_dim=d, q_off=0, k_off=d,
                          v_off=2 * d, status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert torch.equal(q, qkv[:, :d]) and pool[1, 0, 0, 15].any() and not pool[0].any() and not pool[1, :, :, :15].any()


# ---- attention ----------------------------------------------------------------------------------------------------------
def _batch(seed, lengths, nodes, H, G, d, *, chain=False, holes=True, spare_pages=2):
    """Requests with `lengths` cached tokens, the last `nodes` of them drafted; masks that are no trees (any bits), some rows of none."""
    g = gen(seed)
    pages = [-(-n // PAGE) for n in lengths]
    starts = lambda c: i32([sum(c[:k]) for k in range(len(c) + 1)])
    T = sum(nodes)
    words = max(1, -(-max(nodes + [1]) // 64))
    bits = torch.randint(0, 2, (T, words * 64), generator=g, device="cuda").bool()
    own = torch.cat([torch.arange(n, device="cuda") for n in nodes]) if T else torch.zeros(0, dtype=torch.long, device="cuda")
    bits[torch.arange(T, device="cuda"), own] = True
    if holes and T > 2:
        bits[torch.arange(1, T, 5, device="cuda")] = False
    tree = (bits.view(T, words, 64).long() << torch.arange(64, device="cuda")).sum(-1)
    pool = normal(g, sum(pages) + spare_pages, 2, G, PAGE, d)
    return dict(q=normal(g, T, H * d), out=torch.full((T, H * d), 7.0, dtype=torch.bfloat16, device="cuda"), kv_pool=pool, qo_indptr=starts(nodes),
                kv_indptr=starts(pages), kv_indices=torch.randperm(sum(pages) + spare_pages, generator=g, device="cuda")[:sum(pages)].to(torch.int32),
                kv_last_page_len=i32([n - (c - 1) * PAGE if c else 0 for n, c in zip(lengths, pages)]), tree=None if chain else tree, q_heads=H,
                workspace=torch.full_like(ops.tree_workspace(q_heads=H, kv_heads=G, head_dim=d), 255))


def _want(b, sm_scale=None):
    c = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in b.items() if k not in ("out", "workspace")}
    return ref.attn_tree(c.pop("q"), c.pop("kv_pool"), sm_scale=sm_scale, **c)


def _near(out, want, size, rows=None):
    got = out.detach().double().cpu().reshape(want.shape)
    off = (got - want).abs()
    limit = want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -10)
    if rows is not None:
        off, limit = off[rows], limit[rows]
    bad = ~(off <= limit)
    assert not bad.any(), "%d of %d off, worst %.4f" % (int(bad.sum()), bad.numel(), float((off / limit.clamp_min(1e-30))[bad].max()))


HEADS = [(1, 1, 64), (8, 1, 128), (32, 8, 128), (9, 3, 64), (28, 4, 128), (16, 1, 64), (40, 1, 128), (128, 1, 128)]


@pytest.mark.parametrize("H,G,d", HEADS)
@pytest.mark.parametrize("lengths,nodes", [([1], [1]), ([2, 5], [2, 1]), ([16, 17, 40], [1, 1, 3]), ([128, 129, 127], [5, 4, 6]), ([300, 1, 77], [0, 1, 20])])
def test_attention_of_short_contexts(H, G, d, lengths, nodes):
    b = _batch(3, lengths, nodes, H, G, d)
    status = ops.new_status()
    ops.attn_tree(**b, status=status)
    ops.check_status(status)
    _near(b["out"], *_want(b))


@pytest.mark.parametrize("H,G,d,lengths,nodes", [
    (32, 8, 128, [2000], [26]), (32, 8, 128, [700, 64, 1500, 33, 410], [5, 64, 1, 33, 12]), (64, 8, 128, [900, 900], [64, 40]), (12, 12, 64, [1000] * 3, [1, 129, 128]),
    (16, 1, 128, [5000], [70]), (24, 8, 64, [333, 4000], [200, 1]), (4, 1, 64, [600], [512]), (40, 10, 128, [130] * 30, [3] * 30), (2, 2, 128, [3000, 16], [127, 16]),
    (2, 1, 128, [1] * 700, [1] * 700), (8, 8, 64, [20000], [1])])
@pytest.mark.parametrize("chain", [False, True])
def test_attention(H, G, d, lengths, nodes, chain):
    b = _batch(len(lengths) + H, lengths, nodes, H, G, d, chain=chain)
    status = ops.new_status()
    ops.attn_tree(**b, status=status)
    ops.check_status(status)
    want, size = _want(b)
    _near(b["out"], want, size)
    assert not b["out"].view(-1, H, d)[(size == 0).all(-1).cuda()].any()           # rows that see nothing: zeros


def test_attention_where_nothing_is_cached_in_front():
    for n in (1, 3, 64, 65, 200):
        b = _batch(n, [n, n], [n, n], 8, 2, 128)
        ops.attn_tree(**b)
        want, size = _want(b)
        _near(b["out"], want, size)
        if n > 2:
            assert (size == 0).any()


def test_attention_of_a_part_of_the_requests_leaves_the_others_alone():
    b = _batch(5, [100, 50, 900, 20], [7, 9, 11, 3], 8, 2, 128)
    ops.attn_tree(**b, req_begin=1, req_count=2)
    want, size = _want(b)
    _near(b["out"], want, size, slice(7, 27))
    assert (b["out"][:7] == 7).all() and (b["out"][27:] == 7).all()
    # rows behind the last request
    b = _batch(5, [100, 50], [7, 9], 8, 2, 128)
    q, out = torch.cat((b["q"], b["q"][:5])), torch.full((21, 1024), 7.0, dtype=torch.bfloat16, device="cuda")
    tree = torch.cat((b["tree"], b["tree"][:5]))
    ops.attn_tree(**{**b, "q": q, "out": out, "tree": tree})
    want, size = _want(b)
    _near(out[:16], want, size)
    assert (out[16:] == 7).all()


def test_attention_of_strided_rows():
    b = _batch(6, [100, 600], [7, 40], 8, 2, 128)
    plain = ops.attn_tree(**b).clone()
    wide_q, wide_o = torch.zeros(47, 1024 + 520, dtype=torch.bfloat16, device="cuda"), torch.full((47, 2048), 7.0, dtype=torch.bfloat16, device="cuda")
    wide_q[:, 8:1032] = b["q"]
    ops.attn_tree(**{**b, "q": wide_q[:, 8:1032], "out": wide_o[:, 512:1536]})
    assert torch.equal(wide_o[:, 512:1536], plain) and (wide_o[:, :512] == 7).all() and (wide_o[:, 1536:] == 7).all()


@pytest.mark.parametrize("sm_scale", [0.01, 1.0, 3.0])
def test_attention_with_another_scale(sm_scale):
    """Weights from nearly even ones to a single one; the scores' error grows with the scale."""
    b = _batch(7, [1200, 40], [20, 40], 8, 2, 128)
    ops.attn_tree(**b, sm_scale=sm_scale)
    want, size = _want(b, sm_scale)
    _near(b["out"], want, size * (1 if sm_scale <= 1 else 1.25))


@pytest.mark.parametrize("num_ctas", [1, 2, 7, 147, 1000])
def test_attention_within_a_budget(num_ctas):
    b = _batch(8, [900, 40, 2000], [20, 33, 64], 8, 2, 128)
    ops.attn_tree(**b, num_ctas=num_ctas)
    _near(b["out"], *_want(b))


def _spoil(b, r, tokens, value, side):
    """Entries of some cached tokens of request r."""
    first = int(b["kv_indptr"][r])
    for t in tokens:
        page = int(b["kv_indices"][first + t // PAGE])
        b["kv_pool"][page, side, :, t % PAGE, 1::7] = value


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3.3e38])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("lengths,nodes,H,G,d", [([300, 90], [20, 40], 8, 2, 128), ([1000], [100], 8, 2, 64), ([130], [130], 4, 4, 128)])
def test_masked_tokens_do_not_reach_a_row(value, side, lengths, nodes, H, G, d):
    """Drafted tokens with odd keys or values: rows that do not see them are as if they were not there."""
    b = _batch(9, lengths, nodes, H, G, d)
    odd = [[n - k + j for j in (0, 2, k - 1)] for n, k in zip(lengths, nodes)]
    clean = ops.attn_tree(**b).clone()
    sees = torch.zeros(sum(nodes), dtype=torch.bool, device="cuda")
    for r, k in enumerate(nodes):
        a = int(b["qo_indptr"][r])
        for j in (0, 2, k - 1):
            sees[a:a + k] |= (b["tree"][a:a + k, j // 64] >> (j % 64) & 1).bool()
        _spoil(b, r, odd[r], value, side)
        # and what lies behind the last token
        last = int(b["kv_last_page_len"][r])
        b["kv_pool"][int(b["kv_indices"][int(b["kv_indptr"][r + 1]) - 1]), :, :, last:] = float("nan")
    b["kv_pool"][-1] = float("nan") if int(b["kv_indices"].max()) < len(b["kv_pool"]) - 1 else b["kv_pool"][-1]
    ops.attn_tree(**b)
    assert torch.equal(b["out"][~sees], clean[~sees]) and int((~sees).sum()) > 3
    seen = b["out"][sees].view(-1, H, d)
    if side == 1 and abs(value) != 3.3e38:
        assert not seen[..., 1::7].isfinite().any()               # they reach those that see them, and there their own columns only
        other = torch.ones(d, dtype=torch.bool, device="cuda")
        other[1::7] = False
        assert torch.equal(seen[..., other], clean[sees].view(-1, H, d)[..., other])
        if value != value:
            assert seen[..., 1::7].isnan().all()
    if side == 0 and value != value:
        assert seen.isnan().all()


@pytest.mark.parametrize("lengths,nodes,H,G,d", [([30000], [64], 32, 8, 128), ([3000, 90], [20, 3], 8, 2, 128), ([5000, 2], [64, 1], 32, 8, 64)])
def test_sums_of_the_largest_values_stay_finite(lengths, nodes, H, G, d):
    """Values up to 2^127 (of either sign, so that what a row's sums pass through is larger than the row), one KV head of them all alike."""
    b = _batch(18, lengths, nodes, H, G, d)
    b["kv_pool"][:, 1] = (b["kv_pool"][:, 1].float().clamp(-4, 4) * 2.0 ** 125).to(torch.bfloat16)
    b["kv_pool"][:, 1, 0] = 2.0 ** 127
    ops.attn_tree(**b)
    _near(b["out"], *_want(b))


def test_rows_that_only_see_minus_infinity():
    b = _batch(10, [1, 2, 20], [1, 1, 1], 2, 1, 64, chain=True)
    b["q"].abs_()
    _spoil(b, 0, [0], -float("inf"), 0)
    _spoil(b, 1, [0], -float("inf"), 0)
    ops.attn_tree(**b)
    assert b["out"][0].isnan().all() and b["out"][1:].isfinite().all()


def test_lists_that_are_none_are_reported():
    good = _batch(11, [100, 50, 70], [5, 6, 7], 8, 2, 128)
    want, size = _want(good)
    cases = [("kv_indices", 3, -1, None), ("kv_indices", 2, 10 ** 6, None), ("kv_last_page_len", 1, 17, 1), ("kv_last_page_len", 1, 0, 1),
             ("kv_indptr", 1, 1000, 0), ("kv_indptr", 2, -3, 1), ("qo_indptr", 1, 100, 0), ("qo_indptr", 3, 10 ** 9, 2), ("kv_indptr", 2, 7, 1)]
    for name, at, value, req in cases:
        b = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in good.items()}
        b[name][at] = value
        status = ops.new_status()
        ops.attn_tree(**b, status=status)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="index"):
            ops.check_status(status)
        if req != 2 and name != "qo_indptr" and (name, at) != ("kv_indptr", 2):
            _near(b["out"], want, size, slice(11, 18))            # the others' rows are right
        if name == "kv_last_page_len":
            assert not b["out"][5:11].any()


def test_more_queries_than_cached_tokens_are_reported():
    b = _batch(12, [3, 50], [3, 6], 8, 2, 128)
    b["kv_last_page_len"][0] = 2
    status = ops.new_status()
    ops.attn_tree(**b, status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert not b["out"][:3].any()
    _near(b["out"], *_want(b))


def test_tokens_behind_the_last_bit_see_the_context_only():
    """A mask of one word, requests of more tokens: token 64 and those behind it are seen by none."""
    b = _batch(13, [200], [100], 4, 1, 128)
    b["tree"] = b["tree"][:, :1].contiguous()
    ops.attn_tree(**b)
    _near(b["out"], *_want(b))


def test_results_do_not_depend_on_the_workspace_or_the_run():
    b = _batch(14, [900, 40, 2000, 333], [20, 33, 64, 1], 32, 8, 128)
    first = ops.attn_tree(**b).clone()
    for fill in (0, 127, 255):
        b["workspace"].fill_(fill)
        b["out"].fill_(1.0)
        assert torch.equal(ops.attn_tree(**b), first)


def test_far_places_in_a_large_pool():
    """Offsets beyond 32 bits: pages at the end of a pool of 4.6 GB and more."""
    G, d = 8, 128
    pages = 72000
    pool = torch.zeros(pages, 2, G, PAGE, d, dtype=torch.bfloat16, device="cuda")
    b = _batch(15, [500, 90], [20, 8], 32, G, d)
    at = pages - 1 - 2 * torch.arange(int(b["kv_indptr"][-1]), device="cuda")
    pool[at] = b["kv_pool"][b["kv_indices"].long()]
    want, size = _want(b)
    ops.attn_tree(**{**b, "kv_pool": pool, "kv_indices": at.to(torch.int32)})
    _near(b["out"], want, size)
    q, qkv = torch.empty(2, 64, dtype=torch.bfloat16, device="cuda"), normal(gen(1), 2, (32 + 2 * G) * d)
    q = torch.empty(2, 32 * d, dtype=torch.bfloat16, device="cuda")
    slots = i32([pages * PAGE - 1, pages * PAGE - 18])
    ops.rope_append_slots(qkv, q, pool, torch.ones(64, device="cuda"), i32([0, 0]), slots, q_heads=32, kv_heads=G, head_dim=d, q_off=0, k_off=32 * d, v_off=40 * d)
    assert torch.equal(pool[-1, 1, :, 15], qkv[0, 40 * d:].view(G, d)) and torch.equal(pool[-2, 0, :, 14], qkv[1, 32 * d:40 * d].view(G, d))
    ops.kv_keep([pool], i32([pages * PAGE - 40, pages * PAGE - 18, pages * PAGE - 1]), i32([[0, 2, -1]]), i32([2]), i32([0, 3]))
    assert torch.equal(pool[-2, 1, :, 14], qkv[0, 40 * d:].view(G, d))


# ---- trees --------------------------------------------------------------------------------------------------------------
def _parents(r, n, roots=1):
    return [-1 if i < roots else r.randint(max(0, i - r.choice([1, 3, 50])), i - 1) for i in range(n)]


@pytest.mark.parametrize("counts,words", [([1], 1), ([0, 3, 64], 1), ([65, 2], 2), ([128, 1, 100], 2), ([129, 200], 4), ([512, 0, 300], 8), ([70], 3), ([5] * 200, 1)])
@pytest.mark.parametrize("roots", [1, 3])
def test_masks(counts, words, roots):
    r = random.Random(sum(counts))
    parents = [p for n in counts for p in _parents(r, n, roots)]
    if counts == [512, 0, 300] and roots == 1:
        parents = list(range(-1, 511)) + parents[512:]            # as deep as it gets
    qo = [sum(counts[:k]) for k in range(len(counts) + 1)]
    first = [r.randint(0, 10 ** 6) for _ in counts]
    positions = i32([first[k] + 7 * (i > 0) for k, n in enumerate(counts) for i in range(n)] + [5, 6])
    mask = torch.full((qo[-1], words), 3, dtype=torch.int64, device="cuda")
    status = ops.new_status()
    assert ops.tree_masks(i32(parents), i32(qo), mask, positions=positions, status=status) is mask
    ops.check_status(status)
    want, depth = ref.tree_masks(torch.tensor(parents), torch.tensor(qo), words)
    assert torch.equal(mask.cpu(), want)
    assert positions.tolist() == [first[k] + int(depth[qo[k] + i]) for k, n in enumerate(counts) for i in range(n)] + [5, 6]


def test_masks_report_what_is_no_tree():
    for parents, at in (([-1, 0, 2, 0], 2), ([-1, 0, 0, 7], 3), ([-2, 0, 0, 0], 0), ([-1, 0, 0, 3], 3)):
        mask, status = torch.zeros(4, 1, dtype=torch.int64, device="cuda"), ops.new_status()
        ops.tree_masks(i32(parents), i32([0, 4]), mask, status=status)
        with pytest.raises(RuntimeError, match="index"):
            ops.check_status(status)
        parents[at] = -1
        assert torch.equal(mask.cpu(), ref.tree_masks(torch.tensor(parents), torch.tensor([0, 4]), 1)[0])
    # more tokens than bits
    mask, status, positions = torch.full((70, 1), 9, dtype=torch.int64, device="cuda"), ops.new_status(), i32([40] * 70)
    ops.tree_masks(i32(list(range(-1, 69))), i32([0, 70]), mask, positions=positions, status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert not mask[64:].any() and mask[63, 0] == -1 and positions.tolist() == [40 + i for i in range(64)] + [40] * 6


@pytest.mark.parametrize("counts,places", [([1], 1), ([0, 1, 5], 4), ([64, 64, 3], 64), ([512, 100], 512), ([40] * 37, 5), ([300], 2), ([30], 0)])
def test_accept(counts, places):
    r = random.Random(places)
    qo = [sum(counts[:k]) for k in range(len(counts) + 1)]
    parents = [p for n in counts for p in _parents(r, n)]
    tokens = [r.randint(0, 3) for _ in parents]
    targets = [r.randint(0, 3) for _ in parents]
    if counts == [512, 100]:
        parents, tokens, targets = list(range(-1, 511)) + parents[512:], [1] * 612, [1] * 612
    R = len(counts)
    path, status = torch.full((R, places), 9, dtype=torch.int32, device="cuda"), ops.new_status()
    n, following, dropped = (torch.full((R,), 9, dtype=torch.int32, device="cuda") for _ in range(3))
    ops.tree_accept(i32(tokens), i32(parents), i32(targets), i32(qo), path, n, following, dropped=dropped, status=status)
    ops.check_status(status)
    want = ref.tree_accept(torch.tensor(tokens), torch.tensor(parents), torch.tensor(targets), torch.tensor(qo), places)
    assert path.tolist() == [p + [-1] * (places - len(p)) for p in want[0]] and n.tolist() == [len(p) for p in want[0]]
    assert following.tolist() == want[1] and dropped.tolist() == want[2]


@pytest.mark.parametrize("counts,layers,G,d", [([1], 1, 1, 64), ([5, 0, 64], 3, 8, 128), ([200, 512], 2, 3, 64), ([30] * 20, 65, 1, 128), ([40], 1, 12, 256)])
def test_keep(counts, layers, G, d):
    r, g = random.Random(layers), gen(layers)
    qo = [sum(counts[:k]) for k in range(len(counts) + 1)]
    pages = qo[-1] // PAGE + 2
    pools = [normal(g, pages, 2, G, PAGE, d) for _ in range(layers)]
    slots = torch.randperm(pages * PAGE, generator=g, device="cuda")[:qo[-1]].to(torch.int32)
    paths = [[0] + sorted(r.sample(range(1, n), r.randint(0, n - 1))) if n else [] for n in counts]
    if counts[0] == 5:
        paths[2] = list(range(64))[:1] + list(range(2, 64))       # all move by one place
    places = max(len(p) for p in paths) + 2
    path = i32([p + [-1] * (places - len(p)) for p in paths])
    want = [p.clone() for p in pools]
    for w in want:
        ref.kv_keep(w, slots, paths, torch.tensor(qo))
    status = ops.new_status()
    ops.kv_keep(pools, slots, path, i32([len(p) for p in paths]), i32(qo), status=status)
    ops.check_status(status)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


@pytest.mark.parametrize("path,counts,slots,qo", [([[0, 0, 2]], [3], [0, 1, 2], [0, 3]), ([[0, 3, -1]], [2], [0, 1, 2], [0, 3]), ([[0, 2, -1]], [4], [0, 1, 2], [0, 3]),
                                                  ([[0, 2, -1]], [-1], [0, 1, 2], [0, 3]), ([[0, 2, -1]], [2], [0, 1, 99], [0, 3]), ([[0, 2, -1]], [2], [0, -1, 2], [0, 3]),
                                                  ([[0, 2, -1]], [2], [0, 1, 2], [0, 4]), ([[0, 2, -1]], [2], [0, 1, 2], [2, 1])])
def test_keep_reports_what_it_cannot_move(path, counts, slots, qo):
    pool = normal(gen(3), 1, 2, 1, PAGE, 64)
    before, status = pool.clone(), ops.new_status()
    ops.kv_keep([pool], i32(slots), i32(path), i32(counts), i32(qo), status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    if path[0][1] == 0:
        before[0, :, :, 1] = before[0, :, :, 1]                   # place 1 is left, place 2 has its own
    assert torch.equal(pool, before)


def test_keep_of_no_pools():
    ops.kv_keep([], i32([0]), i32([[0]]), i32([1]), i32([0, 1]))


# ---- refusals -------------------------------------------------------------------------------------------------------------
def _arguments():
    b = _batch(1, [40, 20], [3, 2], 4, 2, 64)
    t, li = ops.page_tables(3, 4, 9), ops.batch_lists(2, 6, 8)
    d = 64
    rope = dict(qkv=normal(gen(0), 5, 8 * d), q_out=torch.zeros(5, 4 * d, dtype=torch.bfloat16, device="cuda"), kv_pool=b["kv_pool"], inv_freq=torch.ones(32, device="cuda"),
                positions=i32([0] * 5), slots=i32([0, 1, 2, 3, 4]), q_heads=4, kv_heads=2, head_dim=d, q_off=0, k_off=4 * d, v_off=6 * d)
    masks = dict(parents=i32([-1, 0, 0, -1, 0]), qo_indptr=i32([0, 3, 5]), mask=torch.zeros(5, 1, dtype=torch.int64, device="cuda"), positions=i32([0] * 5))
    accept = dict(tokens=i32([0] * 5), parents=masks["parents"], targets=i32([0] * 5), qo_indptr=masks["qo_indptr"], path=torch.zeros(2, 3, dtype=torch.int32, device="cuda"),
                  counts=i32([0, 0]), next_tokens=i32([0, 0]), dropped=i32([0, 0]))
    keep = dict(kv_pools=[b["kv_pool"].clone(), b["kv_pool"].clone()], slots=i32([0, 1, 2, 3, 4]), path=i32([[0, 2, -1], [0, 1, -1]]), counts=i32([2, 2]), qo_indptr=i32([0, 3, 5]))
    grow = dict(tables=t, rows=i32([0, 1]), new_tokens=i32([3, 3]), lists=li)
    trim = dict(tables=t, rows=i32([0, 1]), dropped=i32([0, 0]))
    return {"attend": (ops.attn_tree, b), "rope": (ops.rope_append_slots, rope), "masks": (ops.tree_masks, masks), "accept": (ops.tree_accept, accept),
            "keep": (ops.kv_keep, keep), "grow": (ops.tables_grow, grow), "trim": (ops.tables_trim, trim)}


def test_the_arguments_below_are_taken():
    for call, args in _arguments().values():
        call(**args)
    torch.cuda.synchronize()


def _with(args, name, value):
    import dataclasses

    if "." in name:
        of, field = name.split(".")
        return {**args, of: dataclasses.replace(args[of], **{field: value(getattr(args[of], field))})}
    return {**args, name: value(args[name])}


BAD = [("attend", "q", lambda x: x.float()), ("attend", "q", lambda x: x.t().contiguous().t()), ("attend", "q", lambda x: x[:, :128]), ("attend", "q", lambda x: x.cpu()),
       ("attend", "q", lambda x: x.view(5, 4, 64)), ("attend", "q", lambda x: x[:1].expand(5, 256)), ("attend", "out", lambda x: x[:4]), ("attend", "kv_pool", lambda x: x.float()),
       ("attend", "kv_pool", lambda x: x[:, :1]), ("attend", "kv_pool", lambda x: x.transpose(2, 3)), ("attend", "qo_indptr", lambda x: x.long()), ("attend", "qo_indptr", lambda x: x[:2]),
       ("attend", "kv_indptr", lambda x: x[:2]), ("attend", "tree", lambda x: x.int()), ("attend", "tree", lambda x: x[:4]), ("attend", "tree", lambda x: x.expand(5, 9).contiguous()),
       ("attend", "tree", lambda x: x[:, :0]), ("attend", "q_heads", lambda x: 3), ("attend", "q_heads", lambda x: 2), ("attend", "workspace", lambda x: x[:1000]),
       ("attend", "workspace", lambda x: None), ("attend", "workspace", lambda x: x[16:]), ("attend", "q", lambda x: torch.zeros(5, 258, dtype=x.dtype, device="cuda")[:, :256]),
       ("rope", "qkv", lambda x: x[:, :500]), ("rope", "qkv", lambda x: x.float()), ("rope", "q_out", lambda x: x[:4]), ("rope", "q_out", lambda x: x.float()), ("rope", "kv_pool", lambda x: x[..., :32].contiguous()),
       ("rope", "inv_freq", lambda x: torch.ones(33, device="cuda")), ("rope", "inv_freq", lambda x: x[:0]), ("rope", "inv_freq", lambda x: x.double()), ("rope", "positions", lambda x: x[:4]),
       ("rope", "slots", lambda x: x.long()), ("rope", "q_heads", lambda x: 5), ("rope", "kv_heads", lambda x: 1), ("rope", "k_off", lambda x: 4), ("rope", "v_off", lambda x: -8),
       ("rope", "head_dim", lambda x: 128), ("masks", "mask", lambda x: x.int()), ("masks", "mask", lambda x: x[:4]), ("masks", "mask", lambda x: x.view(-1)),
       ("masks", "mask", lambda x: torch.zeros(5, 9, dtype=torch.int64, device="cuda")), ("masks", "positions", lambda x: x[:4]), ("masks", "qo_indptr", lambda x: x[:0]),
       ("accept", "path", lambda x: x[:1]), ("accept", "path", lambda x: x.t()), ("accept", "counts", lambda x: x[:1]), ("accept", "targets", lambda x: x[:4]), ("accept", "tokens", lambda x: x.long()),
       ("keep", "kv_pools", lambda x: x[0]), ("keep", "kv_pools", lambda x: [x[0], x[1][:3]]), ("keep", "kv_pools", lambda x: [x[0], None]), ("keep", "kv_pools", lambda x: [x[0], x[0]]),
       ("keep", "kv_pools", lambda x: [x[0], x[1].float()]), ("keep", "path", lambda x: x.view(-1)), ("keep", "counts", lambda x: x[:1]),
       ("grow", "rows", lambda x: x[:1]), ("grow", "rows", lambda x: i32([0] * 4097)), ("grow", "tables.table", lambda x: x.long()), ("grow", "tables.table", lambda x: x[:2]),
       ("grow", "tables.lengths", lambda x: x[:2]), ("grow", "lists.qo_indptr", lambda x: x[:2]), ("grow", "lists.slots", lambda x: x[:5]), ("grow", "lists.positions", lambda x: x.long()),
       ("trim", "dropped", lambda x: x[:1]), ("trim", "tables.free_count", lambda x: i32([1, 1])), ("trim", "tables.ticket", lambda x: i32([]))]


@pytest.mark.parametrize("op,name,value", BAD, ids=["%s-%s-%d" % (c[0], c[1], i) for i, c in enumerate(BAD)])
def test_bad_arguments_are_refused(op, name, value):
    call, args = _arguments()[op]
    with pytest.raises(RuntimeError):
        call(**_with(args, name, value))


def _over(t, dtype, n, first=0):
    return t.view(-1).view(torch.uint8).view(dtype)[first:first + n]


OVERLAPS = [("attend", "out", lambda a: a["q"]), ("attend", "out", lambda a: _over(a["kv_pool"], torch.bfloat16, 1280).view(5, 256)),
            ("attend", "tree", lambda a: _over(a["workspace"], torch.int64, 5).view(5, 1)), ("attend", "qo_indptr", lambda a: _over(a["out"], torch.int32, 3)),
            ("attend", "status", lambda a: a["kv_indptr"]), ("rope", "q_out", lambda a: a["qkv"].view(-1)[:1280].view(5, 256)), ("rope", "slots", lambda a: _over(a["kv_pool"], torch.int32, 5)),
            ("rope", "qkv", lambda a: _over(a["kv_pool"], torch.bfloat16, 2560).view(5, 512)), ("masks", "positions", lambda a: a["parents"]), ("masks", "parents", lambda a: _over(a["mask"], torch.int32, 5)),
            ("accept", "counts", lambda a: a["next_tokens"]), ("accept", "path", lambda a: _over(a["tokens"], torch.int32, 5).view(-1)[:3].view(1, 3).expand(2, 3)),
            ("accept", "dropped", lambda a: a["targets"][:2]), ("keep", "path", lambda a: _over(a["kv_pools"][1], torch.int32, 6).view(2, 3)), ("keep", "status", lambda a: a["counts"]),
            ("keep", "kv_pools", lambda a: [a["kv_pools"][0], a["kv_pools"][0]])]


@pytest.mark.parametrize("op,name,value", OVERLAPS, ids=["%s-%s-%d" % (c[0], c[1], i) for i, c in enumerate(OVERLAPS)])
def test_overlaps_are_refused(op, name, value):
    call, args = _arguments()[op]
    with pytest.raises(RuntimeError):
        call(**{**args, name: value(args)})


def test_overlapping_tables_are_refused():
    call, args = _arguments()["grow"]
    t, li = args["tables"], args["lists"]
    for name, value in (("lists.slots", t.table.view(-1)[:6]), ("lists.positions", li.slots), ("lists.kv_indptr", li.qo_indptr), ("tables.lengths", t.free_pages[:3]), ("tables.ticket", t.free_count)):
        with pytest.raises(RuntimeError, match="overlap"):
            call(**_with(args, name, lambda _: value))
    with pytest.raises(RuntimeError, match="overlap"):
        call(**{**args, "rows": t.lengths[:2]})


# ---- streams, graphs, a run of all of them ------------------------------------------------------------------------------
def test_another_stream():
    b = _batch(16, [900, 300], [20, 64], 32, 8, 128)
    want = ops.attn_tree(**b).clone()
    s = torch.cuda.Stream()
    out, ws = torch.empty_like(b["out"]), torch.empty_like(b["workspace"])
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            ops.attn_tree(**{**b, "out": out, "workspace": ws})
    for _ in range(3):
        ops.attn_tree(**b)                                        # both at once
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(b["out"], want)


class Loop:
    """Requests whose tokens are known; every step drafts trees around what comes next, checks them, and keeps what is right."""

    H, G, D, VOCAB, LAYERS = 8, 2, 64, 50, 2

    def __init__(self, lengths, capacity, seed):
        g, self.r = gen(seed), random.Random(seed)
        self.truth = [[self.r.randrange(self.VOCAB) for _ in range(400)] for _ in lengths]
        self.done = list(lengths)                                 # tokens in the cache; truth[done] is sure, and not cached yet
        R, self.capacity = len(lengths), capacity
        self.embed = [normal(g, self.VOCAB, (self.H + 2 * self.G) * self.D) for _ in range(self.LAYERS)]
        self.pools = [torch.full((R * 26, 2, self.G, PAGE, self.D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(self.LAYERS)]
        self.tables, self.lists = ops.page_tables(R + 2, 26, R * 26), ops.batch_lists(R, capacity, R * 26)
        self.rows = i32([self.r.sample(range(R + 2), R)]).view(-1)
        self.inv, self.factor = ops.rope_frequencies(self.D // 2, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
        T = capacity
        self.q, self.out = ([torch.zeros(T, self.H * self.D, dtype=torch.bfloat16, device="cuda") for _ in range(self.LAYERS)] for _ in range(2))
        self.mask, self.ws = torch.zeros(T, 1, dtype=torch.int64, device="cuda"), ops.tree_workspace(q_heads=self.H, kv_heads=self.G, head_dim=self.D)
        self.new, self.tokens, self.parents, self.targets = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (R, T, T, T))
        self.path, self.status = torch.zeros(R, 12, dtype=torch.int32, device="cuda"), ops.new_status()
        self.counts, self.next, self.dropped = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(3))

    def step(self):
        """The GPU's part: fixed sizes, nothing that waits."""
        li, at = self.lists, dict(status=self.status)
        ops.tables_grow(self.tables, self.rows, self.new, li, **at)
        ops.tree_masks(self.parents, li.qo_indptr, self.mask, positions=li.positions, **at)
        for l in range(self.LAYERS):
            qkv = self.embed[l][self.tokens.long()]
            d, hd = self.D, self.H * self.D
            ops.rope_append_slots(qkv, self.q[l], self.pools[l], self.inv, li.positions, li.slots, q_heads=self.H, kv_heads=self.G, head_dim=d, q_off=0, k_off=hd,
                                  v_off=hd + self.G * d, interleaved=True, factor=self.factor, **at)
            ops.attn_tree(self.q[l], self.out[l], self.pools[l], li.qo_indptr, li.kv_indptr, li.kv_indices, li.kv_last_page_len, self.mask, q_heads=self.H, workspace=self.ws, **at)
        ops.tree_accept(self.tokens, self.parents, self.targets, li.qo_indptr, self.path, self.counts, self.next, dropped=self.dropped, **at)
        ops.kv_keep(self.pools, li.slots, self.path, self.counts, li.qo_indptr, **at)
        ops.tables_trim(self.tables, self.rows, self.dropped, **at)

    def draft(self, prompt=False):
        tokens, parents, targets, new, self.right = [], [], [], [], []
        for k, truth in enumerate(self.truth):
            n0, at = len(tokens), self.done[k]
            if prompt:                                            # a chain of all that is sure
                chain = truth[:at]
                tokens += chain
                parents += list(range(-1, at - 1))
                targets += truth[1:at + 1]
                new.append(at)
                self.right.append(None)
                continue
            place, depth, branch = [-1], [0], [0]                 # of each node: parent, depth, whether it is right; node 0 is sure
            own = [truth[at]]
            for i in range(1, self.r.randint(1, 9)):
                p = self.r.randint(max(0, i - 3), i - 1)
                token = truth[at + depth[p] + 1] if self.r.random() < 0.6 else self.r.randrange(self.VOCAB)
                place.append(p)
                depth.append(depth[p] + 1)
                own.append(token)
            tokens += own
            parents += place
            targets += [truth[at + d + 1] for d in depth]         # what comes next, at that depth
            new.append(len(own))
            kept, node = [0], 0
            while True:
                fits = [i for i in range(node + 1, len(own)) if place[i] == node and own[i] == truth[at + depth[node] + 1]]
                if not fits or len(kept) == 12:
                    break
                node = fits[0]
                kept.append(node)
            self.right.append(kept)
        n = len(tokens)
        assert n <= self.capacity
        pad = [0] * (self.capacity - n)
        for x, v in ((self.tokens, tokens + pad), (self.parents, parents + pad), (self.targets, targets + pad), (self.new, new)):
            x.copy_(i32(v))

    def check(self):
        ops.check_status(self.status)
        scale = self.D ** -0.5
        lens = self.tables.lengths[self.rows.long()].tolist()
        for k, truth in enumerate(self.truth):
            kept = self.right[k]
            assert self.counts[k].item() == len(kept) and self.path[k, :len(kept)].tolist() == kept
            assert self.next[k].item() == truth[self.done[k] + len(kept)]
            n = self.done[k] + len(kept)
            assert lens[k] == n
            pages = self.tables.table[int(self.rows[k]), :-(-n // PAGE)].long()
            ids = torch.tensor(truth[:n], device="cuda")
            for l in range(self.LAYERS):
                # the cache holds exactly the right tokens, and their rows are attention over what lies in front of them
                x = self.embed[l][ids]
                hd, gd = self.H * self.D, self.G * self.D
                key = ref.rope_layout(x[:, hd:hd + gd].view(n, self.G, self.D), torch.arange(n, device="cuda"), self.inv, True, self.factor)
                got = self.pools[l][pages].permute(1, 0, 3, 2, 4).reshape(2, -1, self.G, self.D)[:, :n]
                assert ((got[0].double() - key).abs() <= key.abs() * 2.0 ** -8 + 2.0 ** -17).all() and torch.equal(got[1], x[:, hd + gd:].view(n, self.G, self.D))
                first = int(self.lists.qo_indptr[k])
                rows = torch.tensor(kept, device="cuda") + first
                for i, row in enumerate(rows.tolist()):
                    m = self.done[k] + i + 1
                    q = self.q[l][row].double().view(self.G, -1, self.D)
                    p = torch.softmax(torch.einsum("ghd,ngd->ghn", q, got[0][:m].double()) * scale, -1)
                    v = got[1][:m].double()
                    want, size = torch.einsum("ghn,ngd->ghd", p, v), torch.einsum("ghn,ngd->ghd", p, v.abs())
                    off = (self.out[l][row].double().view(want.shape) - want).abs()
                    assert (off <= want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -10)).all()
            self.done[k] = n
        used = sum(-(-n // PAGE) for n in self.done)
        assert self.tables.free_count.item() == len(self.tables.free_pages) - used


def _begun(loop):
    """The prompts, as chains."""
    loop.draft(prompt=True)
    li = loop.lists
    ops.tables_grow(loop.tables, loop.rows, loop.new, li, status=loop.status)
    for l in range(loop.LAYERS):
        hd = loop.H * loop.D
        ops.rope_append_slots(loop.embed[l][loop.tokens.long()], loop.q[l], loop.pools[l], loop.inv, li.positions, li.slots, q_heads=loop.H, kv_heads=loop.G, head_dim=loop.D,
                              q_off=0, k_off=hd, v_off=hd + loop.G * loop.D, interleaved=True, factor=loop.factor, status=loop.status)
    ops.check_status(loop.status)


def test_two_calls_at_once():
    """Two streams, a workspace each, one of them with a captured graph: as one after the other."""
    torch.cuda.synchronize()
    calls = [_batch(30, [900, 300, 2000], [60, 64, 33], 32, 8, 128), _batch(31, [700] * 20, [5] * 20, 32, 8, 128), _batch(32, [1500, 40], [100, 3], 16, 2, 64)]
    want = [ops.attn_tree(**b).clone() for b in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_tree(**calls[0])
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    for b in calls:
        b["out"].fill_(1.0)
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(one):
            graph.replay()
            ops.attn_tree(**calls[2])
        with torch.cuda.stream(other):
            ops.attn_tree(**calls[1])
    torch.cuda.synchronize()
    for b, w in zip(calls, want):
        assert torch.equal(b["out"], w)


@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_all_of_them(captured):
    loop = Loop([1, 30, 16, 100, 47], 256, 4)
    _begun(loop)
    run = loop.step
    if captured:
        loop.new.zero_()                                          # warm-up and capture change nothing
        loop.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loop.step()
        run = graph.replay
    for _ in range(12):
        loop.draft()
        run()
        loop.check()


@pytest.mark.parametrize("H,G,d", [(32, 8, 128), (24, 8, 64)])
def test_many_requests_give_the_same_again(H, G, d):
    """Several items to a CTA, cut anywhere: places of the ring are taken again while the tiles before are still on their way."""
    r = random.Random(2)
    nodes = [r.randint(1, 5) for _ in range(64)]
    b = _batch(17, [r.randint(200, 4000) + n for n in nodes], nodes, H, G, d, chain=True)
    first = ops.attn_tree(**b).clone()
    for _ in range(10):
        b["out"].fill_(7)
        assert torch.equal(ops.attn_tree(**b), first)
    starts = b["qo_indptr"].tolist()
    want, size = _want({**b, "kv_last_page_len": b["kv_last_page_len"][:9]})
    _near(first[:starts[9]], want[:starts[9]], size[:starts[9]])
