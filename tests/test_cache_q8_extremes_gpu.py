"""The 8-bit KV cache at the ends of its numbers' range, against plain forms in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from nanoflow_b200 import ops
from nanoflow_b200.ops import reference as ref

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = pytest.mark.parametrize("kind", [E4M3, INT8], ids=["e4m3", "int8"])
DIM = 128


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _append(qkv, kind, positions=None, **kw):
    """Tokens of one request with one head of queries, keys and values: (q, numbers, scales) of keys and of values by token."""
    T = qkv.shape[0]
    positions = range(T) if positions is None else positions
    pages = max(positions) // 16 + 1
    pool, scale = ops.kv_pool_q8(pages, 1, DIM, kind)
    q = torch.full((T, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    st = ops.new_status()
    ops.rope_append_q8(qkv, q, pool, scale, torch.ones(DIM // 2, device="cuda"), _i32(list(positions)), _i32([0] * T), _i32([0, pages]),
                       _i32(list(range(pages))), q_heads=1, kv_heads=1, head_dim=DIM, q_off=0, k_off=DIM, v_off=2 * DIM, status=st, **kw)
    ops.check_status(st)
    at = [(p // 16, p % 16) for p in positions]
    pick = lambda t, side: torch.stack([t[a, side, 0, b] for a, b in at])
    numbers = pool.view(torch.int8)
    return q, [pick(numbers, side).view(kind).cpu().double() for side in (0, 1)], [pick(scale, side).cpu().double() for side in (0, 1)], (pool, scale)


def _check_vectors(y, numbers, scale, kind):
    """Half a step of the number's type; the scale's and the quotient's fp32 roundings, the angles' and the norms' sums: 2^-19 of the
    largest entry."""
    most = y.abs().amax(-1, keepdim=True)
    assert bool(((scale[:, None] * ref.Q8_LARGEST[kind] - most).abs() <= 2.0 ** -19 * most).all())
    half = 0.5 * scale[:, None] if kind == INT8 else torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * scale[:, None])
    err = (numbers * scale[:, None] - y).abs()
    assert bool((err <= half + 2.0 ** -19 * most).all()), float((err / most).max())


LARGEST_BF16 = (2 - 2.0 ** -7) * 2.0 ** 127


@KINDS
def test_append_of_the_largest_finite_vectors(kind):
    """Largest entries from 2^125 to the largest of bf16, of either sign, at places of either half: no rotation (position 0) and norms
    whose weights bring keys there."""
    g = torch.Generator().manual_seed(1)
    tops = [2.0 ** 125, 2.0 ** 126, 2.0 ** 126 * (1 + 2.0 ** -7), 2.0 ** 127, -1.5 * 2.0 ** 127, LARGEST_BF16, -LARGEST_BF16]
    for i, top in enumerate(tops):
        x = torch.rand(1, 3 * DIM, generator=g).mul(2).sub(1).double() * 0.9 * abs(top)
        x[0, DIM + 11 * i] = top
        x[0, 2 * DIM + DIM - 1 - 11 * i] = top
        x = x.to(torch.bfloat16).cuda()
        q, numbers, scale, (pool, scales) = _append(x, kind)
        assert torch.equal(q, x[:, :DIM])
        for side in (0, 1):
            _check_vectors(x[:, (1 + side) * DIM:(2 + side) * DIM].double().cpu(), numbers[side], scale[side], kind)
        back = ops.kv_read_q8(pool, scales, _i32([0]))[0, :, 0, 0].double().cpu()
        want = x[0, DIM:].view(2, DIM).double().cpu()
        assert bool(((back - want).abs() <= (2.0 ** -8 + (0.5 / 127 if kind == INT8 else 2.0 ** -4) + 2.0 ** -19) * want.abs().amax(-1, keepdim=True)).all())
        w = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
        normal = torch.randn(1, 3 * DIM, generator=g).to(torch.bfloat16).cuda()
        normal[0, DIM:2 * DIM] = normal[0, DIM:2 * DIM].clamp(-1.5, 1.5)        # (its norm takes 1.5 to less than 2)
        w *= 2.0 ** 126
        _, rk, _ = ref.rope_append_q8(normal.cpu(), torch.ones(DIM // 2), torch.zeros(1), q_heads=1, kv_heads=1, head_dim=DIM, q_off=0, k_off=DIM,
                                      v_off=2 * DIM, k_norm=w.cpu())
        assert 2.0 ** 126 < float(rk.abs().max()) < 2.0 ** 128
        _, numbers, scale, _ = _append(normal, kind, k_norm=w)
        _check_vectors(rk[:, 0], numbers[0], scale[0], kind)


@KINDS
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -120, 1e-6, 3.0])
def test_norms_of_heads_whose_squares_leave_fp32(kind, eps):
    """Entries from 2^-120 to the largest of bf16 in front of the norms of queries and keys, one size to a token, normal ones between
    them (which keep the bits that they have alone)."""
    g = torch.Generator().manual_seed(2)
    sizes = [2.0 ** 60, 2.0 ** 63, 1.0, 2.0 ** 64, 2.0 ** 90, 2.0 ** 120, 2.0 ** 125, 1.0, 2.0 ** -50, 2.0 ** -70, 2.0 ** -75, 2.0 ** -120]
    x = torch.randn(len(sizes), 3 * DIM, generator=g).clamp(-3.9, 3.9)
    x = (x.double() * torch.tensor(sizes, dtype=torch.double)[:, None]).to(torch.bfloat16)
    x[6, DIM] = x[6, 5] = LARGEST_BF16
    assert bool(x.isfinite().all())
    w = [(1 + 0.1 * torch.randn(DIM, generator=g)).to(torch.bfloat16) for _ in range(2)]
    positions = [3 * t for t in range(len(sizes))]
    q, numbers, scale, _ = _append(x.cuda(), kind, positions, q_norm=w[0].cuda(), k_norm=w[1].cuda(), eps=eps)
    rq, rk, rv = ref.rope_append_q8(x, torch.ones(DIM // 2), torch.tensor(positions), q_heads=1, kv_heads=1, head_dim=DIM, q_off=0, k_off=DIM,
                                    v_off=2 * DIM, q_norm=w[0], k_norm=w[1], eps=eps)
    # angles, norms' sums and the rotation in fp32: 2^-20 of the largest entry (and bf16's smallest step, 2^-133)
    err = (q.cpu().double() - rq[:, 0]).abs()
    assert bool((err <= 2.0 ** -8 * rq[:, 0].abs() + 2.0 ** -20 * rq[:, 0].abs().amax(-1, keepdim=True) + 2.0 ** -133).all()), float(err.max())
    seen = rk[:, 0].abs().amax(-1) >= 2.0 ** -79              # (below 2^-80 vectors are zeros)
    _check_vectors(rk[seen, 0], numbers[0][seen], scale[0][seen], kind)
    assert not numbers[0][~seen].any() and not scale[0][~seen].any()
    normal = [2, 7]
    alone = _append(x[normal].cuda(), kind, [positions[t] for t in normal], q_norm=w[0].cuda(), k_norm=w[1].cuda(), eps=eps)
    assert torch.equal(alone[0], q[normal]) and torch.equal(alone[1][0], numbers[0][normal]) and torch.equal(alone[2][0], scale[0][normal])


@KINDS
@pytest.mark.parametrize("size", [2.0 ** 126, 2.0 ** -70])
@pytest.mark.parametrize("lengths,prefix", [([100, 7, 40], 0), ([4000, 7, 333, 50], 0), ([37 * i % 301 for i in range(1, 200)], 0), ([100, 0, 700], 900)])
def test_attention_over_values_at_the_ends_of_the_range(kind, size, lengths, prefix):
    """Values next to the largest of bf16, and next to those that are stored as zeros: sums over tokens leave fp32, results do not."""
    import test_cache_q8_gpu as base

    n, heads, kv_heads = len(lengths), 8, 2
    pages = sum(-(-x // 16) for x in lengths) + -(-prefix // 16) + 1
    pool, scale = base._cache(pages, kv_heads, DIM, kind, spread=0.0)
    scale[:, 1] = scale[:, 1] * (size / (scale[:, 1].max() * ref.Q8_LARGEST[kind] / 3.9))       # the largest value: 3.9 sizes
    pool.view(torch.int8)[:, 1] &= 0x7f          # all of one sign, so that sums grow
    assert float(ref.kv_values_q8(pool, scale, torch.arange(pages)).abs().max()) < 2.0 ** 128
    ptr, idx, last = base._lists(lengths, pages, 3)
    front = torch.arange(-(-prefix // 16), dtype=torch.int32, device="cuda")
    q = torch.randn(n, heads * DIM, device="cuda").to(torch.bfloat16)
    args = (pool, scale, torch.arange(n + 1, dtype=torch.int32, device="cuda"), ptr, idx, last)
    ws = ops.decode_workspace_q8(requests=n, q_heads=heads, kv_heads=kv_heads, head_dim=DIM, prefix_len=prefix)
    out = torch.full_like(q, 3.0)
    ops.attn_decode_shared_q8(q, out, *args, front, prefix, q_heads=heads, req_begin=0, req_count=n, workspace=ws)
    base._check_rows(out, ref.attn_decode_q8(q, *args, q_heads=heads, req_begin=0, req_count=n, prefix_pages=front if prefix else None,
                                             prefix_len=prefix), DIM)
