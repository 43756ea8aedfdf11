"""What the 8-bit cache's calls refuse, and how its work is cut."""
from ctypes import byref, c_longlong, c_void_p

import pytest
import torch

from nanoflow_b200 import ops
from nanoflow_b200.ops import cache_q8 as q8
from nanoflow_b200.ops import reference as ref


def test_pool():
    pool, scale = ops.kv_pool_q8(3, 2, 64, torch.int8, "cpu")
    assert pool.shape == (3, 2, 2, 16, 64) and pool.dtype == torch.int8 and scale.shape == (3, 2, 2, 16) and not scale.any()
    assert ops.kv_pool_q8(3, 2, 64, device="cpu")[0].dtype == torch.float8_e4m3fn
    with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
        ops.kv_pool_q8(3, 2, 64, torch.float16, "cpu")


def test_tensors_that_are_not_on_the_gpu_are_refused():
    pool, scale = ops.kv_pool_q8(3, 2, 64, torch.int8, "cpu")
    one = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 6 * 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_read_q8(pool, scale, one)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rope_append_q8(x, x[:, :128], pool, scale, torch.ones(32), one, one, one, one, q_heads=2, kv_heads=2, head_dim=64, q_off=0, k_off=128,
                           v_off=256)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_q8(x, x, pool, scale, one, one, one, one, q_heads=2, req_begin=0, req_count=1, workspace=one)


def _attn(**kw):
    p = q8.AttnQ8Params(q_heads=8, kv_heads=2, head_dim=128, num_pages=4, num_tokens=3, num_indices=4, req_begin=0, req_count=3, prefix_len=0,
                        kind=0, sm_scale=0.1, num_ctas=0, workspace=4096, workspace_bytes=1 << 40)
    for f in ("q", "out", "kv_pool", "kv_scale", "qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len", "prefix_pages"):
        setattr(p, f, c_void_p(4096))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,rc", [
    (dict(head_dim=96), 3), (dict(head_dim=256), 3), (dict(q_heads=7), 3), (dict(q_heads=34), 3), (dict(kind=2), 3), (dict(kv_heads=0), 3),
    (dict(req_count=-1), 1), (dict(req_begin=-1), 1), (dict(prefix_len=-1), 1), (dict(q=0), 1), (dict(kv_scale=0), 1), (dict(kv_indices=0), 1),
    (dict(workspace=0), 1), (dict(workspace=4100), 1), (dict(workspace_bytes=1000), 1), (dict(q=4104), 1), (dict(kv_pool=4100), 1),
    (dict(num_pages=0), 1), (dict(num_tokens=0), 1), (dict(prefix_len=5, prefix_pages=0), 1), (dict(num_ctas=-2), 1),
    (dict(num_indices=2 ** 30), 1), (dict(req_count=2 ** 28), 1), (dict(prefix_len=2 ** 30, req_count=2 ** 20), 1), (dict(req_begin=2 ** 31 - 2), 1),
    (dict(req_count=0), 0)])
def test_attention_refuses_before_any_launch(change, rc):
    assert ops.lib().nfk_attn_decode_q8(byref(_attn(**change)), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(head_dim=32), 3), (dict(kind=5), 3), (dict(n_pages=-1), 1), (dict(out=4104), 1), (dict(page_ids=0), 1),
                                       (dict(num_pages=0), 1), (dict(n_pages=0), 0)])
def test_read_refuses_before_any_launch(change, rc):
    p = q8.KvReadQ8Params(4096, 4096, 4096, 4096, 2, 2, 64, 4, 0, 0)
    for k, v in change.items():
        setattr(p, k, v)
    assert ops.lib().nfk_kv_read_q8(byref(p), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(head_dim=96), 3), (dict(kind=-1), 3), (dict(T=-1), 1), (dict(ld_qkv=1001), 1), (dict(k_off=4), 1),
                                       (dict(q_off=-8), 1), (dict(q_norm=4098), 1), (dict(inv_freq=0), 1), (dict(num_reqs=0), 1), (dict(T=0), 0)])
def test_append_refuses_before_any_launch(change, rc):
    p = q8.RopeAppendQ8Params(ld_qkv=1024, T=1, q_heads=2, kv_heads=1, head_dim=128, num_pages=1, num_reqs=1, num_indices=1, kind=0)
    for f in ("qkv", "q_out", "kv_pool", "kv_scale", "inv_freq", "positions", "token_req", "kv_indptr", "kv_indices"):
        setattr(p, f, c_void_p(4096))
    for k, v in change.items():
        setattr(p, k, v)
    assert ops.lib().nfk_rope_append_q8(byref(p), c_void_p(0)) == rc


def test_workspace_grows_with_the_sizes_and_covers_smaller_calls():
    size = lambda **kw: ops.decode_workspace_q8(**{**dict(requests=4, q_heads=8, kv_heads=2, head_dim=128, device="cpu"), **kw}).numel()
    assert size() == size(requests=500)
    assert size() < size(prefix_len=10) < size(prefix_len=10000) <= size(prefix_len=20000) < size(prefix_len=20000, requests=3000)
    last = 0
    for n in range(1, 3000, 37):
        now = size(prefix_len=777, requests=n)
        assert now >= last
        last = now
    with pytest.raises(RuntimeError, match="unsupported"):
        size(q_heads=9)
    with pytest.raises(RuntimeError, match="unsupported"):
        size(requests=2 ** 24, prefix_len=2 ** 24)


@pytest.mark.parametrize("kv_heads,group,dim", [(1, 4, 128), (1, 16, 64), (2, 3, 128), (8, 4, 128)])
def test_workspace_covers_shorter_prefixes_and_fewer_requests(kv_heads, group, dim):
    """Shorter prefixes are cut into smaller shares, fewer requests into other blocks of rows: the larger call's workspace holds them."""
    size = lambda r, n: ops.decode_workspace_q8(requests=r, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=dim, prefix_len=n, device="cpu").numel()
    lengths = [0, 1, 64, 65, 1984, 1985, 2048, 8000, 8128, 8129, 8192, 19000, 40000]
    for counts in zip(lengths, lengths[1:]):
        assert size(8, counts[0]) <= size(8, counts[1])
    for n in lengths:
        sizes = [size(r, n) for r in (1, 7, 8, 9, 31, 32, 33, 42, 43, 85, 86, 500)]
        assert sizes == sorted(sizes)


def test_quantising_in_the_plain_form():
    x = torch.tensor([[1.0, -2.0, 0.0], [0, 0, 0], [1e-30, 0, 0], [float("inf"), 1, 1], [2.0 ** -79, 0, 0]], dtype=torch.double)
    for dtype, largest in ref.Q8_LARGEST.items():
        n, s = ref.quantise_q8(x, dtype)
        assert float(s[0]) == pytest.approx(2 / largest) and float(n[0, 1].double()) == -largest
        assert s[1] == 0 and s[2] == 0 and bool(s[3].isnan()) and float(s[4]) > 0 and not n[1:4].double().any()
