"""Drafted tokens: masks that are smaller than a request, lists that are larger than a step, scores of any size, lists and paths that
are partly none. Tolerances are those of test_draft_gpu.py, unless a test says more."""
import pytest
import torch

import test_draft_gpu as base
from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref

pytestmark = pytest.mark.gpu


# ---- masks ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("words,tokens", [(1, 64), (1, 65), (2, 300), (3, 192), (3, 193), (3, 200), (3, 256), (3, 700), (4, 257), (5, 320), (5, 400), (6, 390),
                                          (7, 448), (7, 449), (7, 512), (8, 512), (8, 513), (8, 1600)])
@pytest.mark.parametrize("chain", [False, True])
def test_tokens_behind_a_masks_last_bit(words, tokens, chain):
    """They see none of the others, stand at the request's first position, and are reported, however many words the mask has."""
    r = base.random.Random(tokens)
    counts = [5, tokens, 70]
    bits = [min(64 * words, n) for n in counts]
    parents = [p for n in counts for p in (range(-1, n - 1) if chain else base._parents(r, n))]
    qo = [sum(counts[:k]) for k in range(4)]
    mask = torch.full((qo[-1], words), 3, dtype=torch.int64, device="cuda")
    first = [1000, 7, 40]
    positions = base.i32([first[k] for k, n in enumerate(counts) for _ in range(n)])
    status = ops.new_status()
    ops.tree_masks(base.i32(parents), base.i32(qo), mask, positions=positions, status=status)
    if all(b == n for b, n in zip(bits, counts)):
        ops.check_status(status)
    else:
        with pytest.raises(RuntimeError, match="index"):
            ops.check_status(status)
    want, depth = ref.tree_masks(torch.tensor(parents), torch.tensor(qo), words)
    for k, n in enumerate(counts):
        a, b = qo[k], qo[k] + bits[k]
        assert torch.equal(mask[a:b].cpu(), want[a:b]) and positions[a:b].tolist() == [first[k] + d for d in depth[a:b].tolist()]
        for i in (0, bits[k] - 1):
            assert int(mask[a + i, i // 64]) >> (i % 64) & 1              # each sees itself
        assert not mask[b:qo[k + 1]].any() and (positions[b:qo[k + 1]] == first[k]).all()
        assert not want[b:qo[k + 1]].any() and not depth[b:qo[k + 1]].any()


# ---- lists of more requests than a step has -------------------------------------------------------------------------------------
@pytest.mark.parametrize("earlier,step", [([10] * 8, [40, 40]), ([10] * 8, [4, 4]), ([1] * 8, [30, 60, 2]), ([10] * 8, [0, 5]), ([10] * 8, [])])
def test_lists_of_more_requests_than_the_step_has(earlier, step):
    """A step in lists that an earlier one with more requests filled: entries behind its last request are requests of nothing, and rows and
    tokens behind the last one are left alone, as with lists of its own."""
    H, G, d, R, C, T, pages = 8, 2, 64, len(step), 8, 140, 100
    lengths = [100, 33, 16, 5, 47, 64, 1, 200]
    t, _ = base._tables(C, 24, 160, lengths)
    g, r = base.gen(3), base.random.Random(1)
    pool = base.normal(g, 160, 2, G, 16, d)
    q = base.normal(g, T, H * d)
    tokens, targets = (torch.randint(0, 3, (T,), generator=g, device="cuda").to(torch.int32) for _ in range(2))
    parents = base.i32([p for n in step for p in base._parents(r, n)] + [0] * (T - sum(step)))
    lists = ops.batch_lists(C, T, pages)
    everyone = base.i32(list(range(C)))
    ops.tables_grow(t, everyone, base.i32(earlier), lists)
    ops.tables_trim(t, everyone, base.i32(earlier))
    ws = ops.tree_workspace(q_heads=H, kv_heads=G, head_dim=d)

    def run(li, requests):
        out, mask = torch.full((T, H * d), 7.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, 1, dtype=torch.int64, device="cuda")
        path, counts, following, dropped = (torch.full(s, 9, dtype=torch.int32, device="cuda") for s in ((requests, 6), (requests,), (requests,), (requests,)))
        cache, status = pool.clone(), ops.new_status()
        ops.tables_grow(t, everyone[:R], base.i32(step), li, status=status)
        ops.tree_masks(parents, li.qo_indptr, mask, positions=li.positions, status=status)
        ops.attn_tree(q, out, cache, li.qo_indptr, li.kv_indptr, li.kv_indices, li.kv_last_page_len, mask, q_heads=H, workspace=ws, status=status)
        ops.tree_accept(tokens, parents, targets, li.qo_indptr, path, counts, following, dropped=dropped, status=status)
        ops.kv_keep([cache], li.slots, path, counts, li.qo_indptr, status=status)
        ops.tables_trim(t, everyone[:R], base.i32(step), status=status)
        torch.cuda.synchronize()
        return [out, mask, li.positions.clone(), cache, path[:R], counts[:R], following[:R], dropped[:R]], [path[R:], counts[R:], following[R:], dropped[R:]], status

    fitting, _, status = run(ops.batch_lists(R, T, pages), R)
    ops.check_status(status)
    same, behind, status = run(lists, C)
    n = sum(step)
    assert (fitting[0][n:] == 7).all() and (n == 0 or not (fitting[0][:n] == 7).all())
    assert lists.qo_indptr[R:].tolist() == [n] * (C + 1 - R)
    assert lists.kv_indptr[R:].tolist() == [int(lists.kv_indptr[R])] * (C + 1 - R) and not lists.kv_last_page_len[R:].any()
    for a, b in zip(fitting, same):
        assert torch.equal(a, b)
    ops.check_status(status)
    assert [x.unique().tolist() for x in behind] == [[-1], [0], [-1], [0]]


def test_lists_of_a_step_that_does_not_fit_are_empty_to_their_ends():
    t, _ = base._tables(6, 20, 90, [0, 15, 16, 100, 31, 64])
    lists = ops.batch_lists(6, 40, 40)
    ops.tables_grow(t, base.i32([0, 1, 2, 3, 4, 5]), base.i32([3] * 6), lists)
    status = ops.new_status()
    ops.tables_grow(t, base.i32([2, 2]), base.i32([1, 1]), lists, status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert not any(x.any() for x in (lists.qo_indptr, lists.kv_indptr, lists.kv_last_page_len, lists.positions)) and (lists.slots == -1).all()


# ---- scores ---------------------------------------------------------------------------------------------------------------------
SHAPES = [([900, 40, 2000], [20, 33, 64], 8, 2, 128), ([700, 64], [40, 64], 64, 8, 128), ([900, 2, 300], [20, 1, 130], 8, 2, 64)]


@pytest.mark.parametrize("lengths,nodes,H,G,d", SHAPES)
def test_scores_that_grow_from_tile_to_tile(lengths, nodes, H, G, d):
    """The reference moves in every tile, and each tile's weights are formed twice: the same result in every run. (Scores of a tile's best
    tokens are above those of the tiles in front by some 2^4 or more.)"""
    b = base._batch(25, lengths, nodes, H, G, d)
    b["q"].abs_()
    for r, n in enumerate(lengths):
        first = int(b["kv_indptr"][r])
        pages = b["kv_indices"][first:int(b["kv_indptr"][r + 1])].long()
        b["kv_pool"][pages, 0] = (b["kv_pool"][pages, 0].float() * 0.1 + torch.arange(len(pages), device="cuda")[:, None, None, None] * (20.0 / d)).to(torch.bfloat16)
    want, size = base._want(b)
    first = ops.attn_tree(**b).clone()
    # sum |q k| scale is below 250 here, so that scores are off by 2^-24 128 250 < 2^-9, and weights and their sum by as much each
    got = first.double().cpu().reshape(want.shape)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -8)).all()
    for _ in range(20):
        b["out"].fill_(7)
        assert torch.equal(ops.attn_tree(**b), first)


def _whole(b, seed, most=3):
    """Queries and keys of small whole numbers: their products are exact in fp32, scores differ by the scale or not at all."""
    g = base.gen(seed)
    b["q"].copy_(torch.randint(-most, most + 1, b["q"].shape, generator=g, device="cuda"))
    b["kv_pool"][:, 0] = torch.randint(-most, most + 1, b["kv_pool"][:, 0].shape, generator=g, device="cuda").to(torch.bfloat16)
    return b


@pytest.mark.parametrize("sm_scale", [1e3, 3e7, 1e8, 1e9, 3e9, 1e10, 1e12, 1e20, 1e35])
@pytest.mark.parametrize("lengths,nodes,H,G,d", SHAPES)
@pytest.mark.parametrize("num_ctas", [0, 1])
def test_rows_of_large_scores(lengths, nodes, H, G, d, sm_scale, num_ctas):
    """Rows are the mean of the values with the largest score, in items of one piece (a single CTA) and in cut ones. Scores are below 3.4e38 /
    log2(e): products are at most 9 d."""
    b = _whole(base._batch(21, lengths, nodes, H, G, d), 5)
    ops.attn_tree(**b, sm_scale=sm_scale, num_ctas=num_ctas)
    base._near(b["out"], *base._want(b, sm_scale))


@pytest.mark.parametrize("lengths,nodes,H,G,d", SHAPES)
def test_rows_of_scores_far_below_zero(lengths, nodes, H, G, d):
    b = _whole(base._batch(22, lengths, nodes, H, G, d), 6)
    b["q"].abs_()
    b["kv_pool"][:, 0] = -b["kv_pool"][:, 0].abs()
    b["kv_pool"][:, 0, :, :, 0], b["q"][:, ::d] = -1, 1            # (none is zero)
    ops.attn_tree(**b, sm_scale=1e11)
    base._near(b["out"], *base._want(b, 1e11))


@pytest.mark.parametrize("lengths,nodes,H,G,d", SHAPES)
@pytest.mark.parametrize("num_ctas", [0, 1])
def test_rows_of_small_and_large_scores_side_by_side(lengths, nodes, H, G, d, num_ctas):
    """Rows whose scores go from some ten to 1e32, neighbours of one warp among them. Powers of two leave the products exact; where scores of a
    row are some 2^k apart at least (k from 8 on), weights are those of ties; below, scores of 3000 at most are off by 2^-24 of themselves."""
    b = _whole(base._batch(23, lengths, nodes, H, G, d), 7)
    T = sum(nodes)
    k = torch.tensor([0, 2, 8, 16, 19, 20, 21, 22, 24, 30, 40, 60, 100], device="cuda")
    rows = b["q"].view(T, H, d)
    rows *= (2.0 ** k[(torch.arange(T, device="cuda")[:, None] * 5 + torch.arange(H, device="cuda")) % len(k)])[..., None].to(torch.bfloat16)
    ops.attn_tree(**b, sm_scale=0.125, num_ctas=num_ctas)
    base._near(b["out"], *base._want(b, 0.125))


def test_sums_of_the_largest_values_with_large_scores_stay_finite():
    """Scores of 1e8 to 1e12 that are all the same, values of 2^127: the mean is as large, the sum of 3000 of them fp32 does not hold."""
    for scale in (1e6, 1e8, 3e8, 1e9, 1e12):
        b = base._batch(24, [3000, 70], [20, 30], 8, 2, 128)
        b["q"].fill_(1)
        b["kv_pool"][:, 0] = 1
        b["kv_pool"][:, 1] = 2.0 ** 127
        ops.attn_tree(**b, sm_scale=scale)
        base._near(b["out"], *base._want(b, scale))


def test_a_pool_that_is_not_aligned_is_refused_before_anything_moves():
    """The last of more pools than a launch takes."""
    pools = [base.normal(base.gen(k), 1, 2, 1, 16, 64) for k in range(64)]
    pools.append(torch.zeros(2049, dtype=torch.bfloat16, device="cuda")[1:].view(1, 2, 1, 16, 64))
    before = [p.clone() for p in pools]
    with pytest.raises(RuntimeError, match="kv_keep"):
        ops.kv_keep(pools, base.i32([0, 1, 2]), base.i32([[0, 2, -1]]), base.i32([2]), base.i32([0, 3]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, pools))


# ---- columns of one buffer ------------------------------------------------------------------------------------------------------
def test_rows_that_lie_between_other_rows():
    """Queries and outputs as columns of one buffer do not overlap; columns that both have do."""
    b = base._batch(6, [100, 600], [7, 40], 8, 2, 128)
    plain = ops.attn_tree(**b).clone()
    row = 1024
    for q_at, out_at in ((0, row), (row + 8, 0), (8, row + 16)):
        wide = torch.full((47, 2 * row + 64), 7.0, dtype=torch.bfloat16, device="cuda")
        wide[:, q_at:q_at + row] = b["q"]
        before = wide.clone()
        ops.attn_tree(**{**b, "q": wide[:, q_at:q_at + row], "out": wide[:, out_at:out_at + row]})
        before[:, out_at:out_at + row] = plain
        assert torch.equal(wide, before)
    wide = torch.zeros(48, 2 * row + 64, dtype=torch.bfloat16, device="cuda")
    for q, out in ((wide[:47, :row], wide[:47, row - 8:2 * row - 8]), (wide[:47, 8:row + 8], wide[:47, :row]), (wide[:47, :row], wide[1:, :row]),
                   (wide[:47, row + 64:], wide[1:, 80:row + 80]), (wide[:47, :row], wide.view(-1)[row:row + 47 * row].view(47, row))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.attn_tree(**{**b, "q": q, "out": out})


# ---- lists and paths that are partly none -----------------------------------------------------------------------------------------
def test_rows_of_lists_that_are_partly_none():
    """Query lists: requests beside the one that is none keep their rows, and rows of nobody are left as they were."""
    good = base._batch(11, [100, 50, 70], [5, 6, 7], 8, 2, 128)
    want, size = base._want(good)
    for at, value, right in ((1, 100, slice(11, 18)), (1, -1, slice(11, 18)), (3, 10 ** 9, slice(0, 11)), (3, 10, slice(0, 11))):
        b = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in good.items()}
        b["qo_indptr"][at] = value
        status = ops.new_status()
        ops.attn_tree(**b, status=status)
        with pytest.raises(RuntimeError, match="index"):
            ops.check_status(status)
        base._near(b["out"], want, size, right)
        rest = torch.ones(18, dtype=torch.bool, device="cuda")
        rest[right] = False
        assert (b["out"][rest] == 7).all()


@pytest.mark.parametrize("path,counts,slots,moved", [([0, 0, 3, -1], 3, [0, 1, 2, 3], {2: 3}), ([0, 2, 5, 3], 4, [0, 1, 2, 3], {1: 2}),
                                                     ([0, 2, 3, -1], 3, [0, 77, 2, 3], {2: 3}), ([0, -1, 3, 3], 4, [4, 5, 6, 7], {6: 7})])
def test_moves_beside_one_that_is_none_are_made(path, counts, slots, moved):
    pool = base.normal(base.gen(3), 1, 2, 1, 16, 64)
    want, status = pool.clone(), ops.new_status()
    for to, source in moved.items():
        want[0, :, :, to] = pool[0, :, :, source]
    ops.kv_keep([pool], base.i32(slots), base.i32([path]), base.i32([counts]), base.i32([0, 4]), status=status)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status(status)
    assert torch.equal(pool, want)


# ---- tables where the number of threads changes ------------------------------------------------------------------------------------
@pytest.mark.parametrize("R", [256, 257, 300, 512, 767, 768, 769, 800])
def test_tables_of_some_hundred_requests(R):
    base.test_grow_and_trim(R, 0, 90, 20, 3)


# ---- how many tokens a request has, as far as the host knows -----------------------------------------------------------------------
@pytest.mark.parametrize("H,G,d", [(32, 8, 128), (24, 8, 64)])
def test_rows_of_padding_and_of_other_requests_do_not_choose_the_form(H, G, d):
    """Short chains in queries with room for 64 tokens each: with request_tokens, the bits of the call whose queries fit. A part of a batch takes
    the batch's form."""
    nodes = [5, 3, 1, 4] * 5
    b = base._batch(41, [600 + 40 * k for k in range(20)], nodes, H, G, d)
    T = sum(nodes)
    fitting = ops.attn_tree(**b).clone()
    q, out = (torch.full((20 * 64, H * d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q[:T] = b["q"]
    tree = torch.zeros(20 * 64, 1, dtype=torch.int64, device="cuda")
    tree[:T] = b["tree"]
    padded = {**b, "q": q, "out": out, "tree": tree}
    assert torch.equal(ops.attn_tree(**padded, request_tokens=5)[:T], fitting) and (out[T:] == 7).all()
    want, size = base._want(b)
    for tokens in (0, 1, 64, 2 ** 31 - 1):
        base._near(ops.attn_tree(**padded, request_tokens=tokens)[:T], want, size)
    part = ops.attn_tree(**b, req_begin=3, req_count=2, request_tokens=5).clone()
    assert torch.equal(ops.attn_tree(**b, req_begin=3, req_count=2), part)
    a, e = sum(nodes[:3]), sum(nodes[:5])
    base._near(part[a:e], want[a:e], size[a:e])


def test_a_number_of_tokens_that_is_none_is_refused():
    b = base._batch(1, [40, 20], [3, 2], 4, 2, 64)
    for bad in (-1, 2 ** 31, 1.5):
        with pytest.raises(RuntimeError, match="attn_tree|bad argument"):
            ops.attn_tree(**b, request_tokens=bad)
