"""Drafted tokens: frequencies of rotations, and what the calls refuse before any launch."""
from ctypes import byref, c_void_p

import pytest
import torch

from nanoflow_b200 import ops
from nanoflow_b200.ops import draft
from nanoflow_b200.ops import reference as ref


# ---- frequencies -----------------------------------------------------------------------------------------------------
def _theirs(rot_dim, theta, scaling, length, max_position):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    config = LlamaConfig(hidden_size=rot_dim * 4, num_attention_heads=4, head_dim=rot_dim, max_position_embeddings=max_position,
                         rope_parameters={"rope_theta": theta, **scaling})
    if "original_max_position_embeddings" in scaling:
        config.original_max_position_embeddings = scaling["original_max_position_embeddings"]
    return ROPE_INIT_FUNCTIONS[scaling["rope_type"]](config, "cpu", seq_len=length)


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096, "mscale": 1.0, "mscale_all_dim": 0.8, "beta_fast": 24, "beta_slow": 2},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "attention_factor": 1.5, "truncate": False},
    {"rope_type": "dynamic", "factor": 2.0}])
@pytest.mark.parametrize("rot_dim", [32, 64, 128])
@pytest.mark.parametrize("length", [100, 50000])
def test_frequencies(scaling, rot_dim, length):
    theirs, factor = _theirs(rot_dim, 10000.0, scaling, length, 8192)
    inv, out = ops.rope_frequencies(rot_dim, 10000.0, scaling, length=length, max_position=8192, device="cpu")
    assert inv.dtype == torch.float32 and inv.shape == (rot_dim // 2,)
    # theirs are formed in fp32: powers of theta to some 2^-20
    torch.testing.assert_close(inv, theirs.float(), rtol=2.0 ** -19, atol=0)
    assert out == pytest.approx(factor, rel=1e-6)


def test_frequencies_longrope():
    scaling = {"rope_type": "longrope", "original_max_position_embeddings": 4096, "short_factor": [1.0 + i / 32 for i in range(32)],
               "long_factor": [2.0 + i for i in range(32)]}
    plain = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    for length, factors in ((100, "short_factor"), (4096, "short_factor"), (4097, "long_factor")):
        inv, out = ops.rope_frequencies(64, 10000.0, scaling, length=length, max_position=131072, device="cpu")
        torch.testing.assert_close(inv, (plain / torch.tensor(scaling[factors]).double()).float(), rtol=0, atol=0)
        assert out == pytest.approx((1 + 5 / 12) ** 0.5)       # sqrt(1 + ln 32 / ln 4096)


def test_frequencies_without_scaling():
    inv, out = ops.rope_frequencies(128, 500000.0, device="cpu")
    torch.testing.assert_close(inv, ref.rope_inv_freq(128, 500000.0), rtol=0, atol=0)
    assert out == 1.0
    for bad in (dict(rot_dim=7), dict(rot_dim=64, scaling={"rope_type": "other"}), dict(rot_dim=64, scaling={"rope_type": "yarn", "factor": 2.0}),
                dict(rot_dim=64, scaling={"rope_type": "linear"}), dict(rot_dim=64, scaling={"rope_type": "dynamic"}, max_position=4096),
                dict(rot_dim=2, scaling={"rope_type": "dynamic", "factor": 2.0}, max_position=4096), dict(rot_dim=64, theta=1.0), dict(rot_dim=64, theta=-2.0),
                dict(rot_dim=64, scaling={"rope_type": "linear", "factor": 0.0}), dict(rot_dim=64, scaling={"rope_type": "longrope"}, max_position=4096),
                dict(rot_dim=64, scaling={"rope_type": "longrope", "short_factor": [1.0] * 31, "long_factor": [1.0] * 31}, max_position=4096),
                dict(rot_dim=64, scaling={"rope_type": "llama3"}), dict(rot_dim=64, scaling={"rope_type": "yarn", "original_max_position_embeddings": 4096}),
                dict(rot_dim=64, scaling={"rope_type": "yarn", "factor": -4.0, "original_max_position_embeddings": 4096})):
        with pytest.raises(RuntimeError, match="rope_frequencies"):
            ops.rope_frequencies(**{"theta": 10000.0, "device": "cpu", **bad})


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_tensors_that_are_not_on_the_gpu_are_refused():
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    t, li = ops.page_tables(2, 3, 5, "cpu"), ops.batch_lists(2, 4, 6, "cpu")
    pool, x = torch.zeros(2, 2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 192, dtype=torch.bfloat16)
    calls = [lambda: ops.tables_grow(t, i(1), i(1), li), lambda: ops.tables_trim(t, i(1), i(1)),
             lambda: ops.rope_append_slots(x, x[:, :64], pool, torch.ones(32), i(2), i(2), q_heads=1, kv_heads=1, head_dim=64, q_off=0, k_off=64, v_off=128),
             lambda: ops.attn_tree(x[:, :64], x[:, :64], pool, i(2), i(2), i(1), i(1), q_heads=1, workspace=i(1)),
             lambda: ops.tree_masks(i(2), i(2), torch.zeros(2, 1, dtype=torch.int64)),
             lambda: ops.tree_accept(i(2), i(2), i(2), i(2), i(2).view(1, 2), i(1), i(1)), lambda: ops.kv_keep([pool], i(2), i(2).view(1, 2), i(1), i(2))]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_new_tables_and_lists():
    t = ops.page_tables(3, 4, 6, "cpu")
    assert t.table.shape == (3, 4) and not t.table.any() and not t.lengths.any() and t.free_pages.tolist() == [5, 4, 3, 2, 1, 0]
    assert t.free_count.tolist() == [6] and t.ticket.tolist() == [0]
    li = ops.batch_lists(2, 5, 7, "cpu")
    assert [x.numel() for x in (li.qo_indptr, li.kv_indptr, li.kv_indices, li.kv_last_page_len, li.positions, li.token_req, li.slots)] == [3, 3, 7, 2, 5, 5, 5]
    assert li.slots.tolist() == [-1] * 5


def _filled(cls, pointers, values, change):
    p = cls(**values)
    for f in pointers:
        setattr(p, f, c_void_p(4096))
    for k, v in change.items():
        setattr(p, k, v)
    return byref(p)


@pytest.mark.parametrize("change,rc", [(dict(requests=-1), 1), (dict(requests=4097), 1), (dict(max_requests=0), 1), (dict(max_requests=65537), 1),
                                       (dict(max_pages=0), 1), (dict(max_pages=2 ** 27), 1), (dict(num_pages=0), 1), (dict(num_pages=2 ** 27), 1), (dict(table=0), 1),
                                       (dict(ticket=0), 1), (dict(rows=0), 1), (dict(kv_indices=0), 1), (dict(slots=0), 1), (dict(num_tokens=-1), 1),
                                       (dict(num_indices=-1), 1)])
def test_tables_refuse_before_any_launch(change, rc):
    pointers = ("table", "lengths", "free_pages", "free_count", "ticket", "rows", "tokens", "qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len",
                "positions", "token_req", "slots")
    values = dict(requests=1, max_requests=1, max_pages=1, num_pages=1, num_indices=1, num_tokens=1)
    assert ops.lib().nfk_tables_grow(_filled(draft.TablesParams, pointers, values, change), c_void_p(0)) == rc
    if not set(change) & {"kv_indices", "slots", "num_tokens", "num_indices"}:
        assert ops.lib().nfk_tables_trim(_filled(draft.TablesParams, pointers, values, change), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(head_dim=96), 3), (dict(head_dim=256), 3), (dict(T=-1), 1), (dict(T=0), 0), (dict(pairs=0), 1), (dict(pairs=33), 1),
                                       (dict(ld_qkv=129), 1), (dict(k_off=4), 1), (dict(v_off=-8), 1), (dict(slots=0), 1), (dict(inv_freq=0), 1),
                                       (dict(q_out=4104), 1), (dict(kv_pool=4100), 1), (dict(num_pages=2 ** 27), 1), (dict(kv_heads=0), 1)])
def test_rotation_refuses_before_any_launch(change, rc):
    pointers = ("qkv", "q_out", "kv_pool", "inv_freq", "positions", "slots")
    values = dict(ld_qkv=192, T=1, q_heads=1, kv_heads=1, head_dim=64, pairs=32, num_pages=1, k_off=64, v_off=128, factor=1.0)
    assert ops.lib().nfk_rope_slots(_filled(draft.RopeSlotsParams, pointers, values, change), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(head_dim=96), 3), (dict(q_heads=7), 3), (dict(q_heads=258), 3), (dict(kv_heads=0), 3), (dict(req_count=-1), 1), (dict(req_begin=-1), 1),
    (dict(req_count=0), 0), (dict(num_tokens=0), 0), (dict(num_ctas=-1), 1), (dict(q=0), 1), (dict(out=4104), 1), (dict(workspace=4112), 1), (dict(workspace_bytes=1000), 1),
    (dict(tree=4100), 1), (dict(words=0), 1), (dict(words=9), 1), (dict(ld_q=1000), 1), (dict(ld_out=1028), 1), (dict(sm_scale=0.0), 1),
    (dict(sm_scale=2.5e38), 1), (dict(ld_out=2 ** 35 // 3 + 8), 1), (dict(ld_out=2 ** 62), 1), (dict(ld_q=2 ** 40), 1), (dict(sm_scale=float("nan")), 1), (dict(sm_scale=float("inf")), 1), (dict(num_pages=0), 1), (dict(num_pages=2 ** 26), 1), (dict(num_indices=-1), 1), (dict(req_begin=2 ** 31 - 2), 1)])
def test_attention_refuses_before_any_launch(change, rc):
    pointers = ("q", "out", "kv_pool", "qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len", "tree", "workspace")
    values = dict(ld_q=1024, ld_out=1024, q_heads=8, kv_heads=2, head_dim=128, num_pages=4, num_tokens=3, num_indices=4, req_count=3, words=1, sm_scale=0.1,
                  workspace_bytes=1 << 40)
    assert ops.lib().nfk_attn_tree(_filled(draft.AttnTreeParams, pointers, values, change), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(requests=-1), 1), (dict(requests=0), 0), (dict(num_tokens=0), 0), (dict(words=0), 1), (dict(words=9), 1),
                                       (dict(mask=4100), 1), (dict(parents=0), 1)])
def test_masks_refuse_before_any_launch(change, rc):
    values = dict(requests=1, num_tokens=1, words=1)
    assert ops.lib().nfk_tree_masks(_filled(draft.TreeMasksParams, ("parents", "qo_indptr", "mask"), values, change), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(requests=-1), 1), (dict(requests=0), 0), (dict(max_path=-1), 1), (dict(path=0), 1), (dict(counts=0), 1), (dict(tokens=0), 1)])
def test_accept_refuses_before_any_launch(change, rc):
    pointers = ("tokens", "parents", "targets", "qo_indptr", "path", "counts", "next_tokens")
    assert ops.lib().nfk_tree_accept(_filled(draft.TreeAcceptParams, pointers, dict(requests=1, num_tokens=1, max_path=1), change), c_void_p(0)) == rc


@pytest.mark.parametrize("change,rc", [(dict(requests=0), 0), (dict(num_pools=65), 1), (dict(num_pools=-1), 1), (dict(num_pools=0), 0), (dict(num_pools=2), 1),
                                       (dict(head_dim=12), 3), (dict(slots=0), 1), (dict(num_pages=0), 1), (dict(kv_heads=0), 1)])
def test_keep_refuses_before_any_launch(change, rc):
    p = draft.KvKeepParams(num_pools=1, requests=1, num_tokens=1, max_path=1, num_pages=1, kv_heads=1, head_dim=64)
    p.pools[0] = 4096
    for f in ("slots", "path", "counts", "qo_indptr"):
        setattr(p, f, c_void_p(4096))
    for k, v in change.items():
        setattr(p, k, v)
    assert ops.lib().nfk_kv_keep(byref(p), c_void_p(0)) == rc


def test_workspace_goes_by_the_head_size_only():
    size = lambda **kw: ops.tree_workspace(**{**dict(q_heads=8, kv_heads=2, head_dim=128, device="cpu"), **kw}).numel()
    assert size() == size(q_heads=128) > size(head_dim=64) > 0
    for bad in (dict(head_dim=96), dict(q_heads=9), dict(q_heads=258), dict(kv_heads=0)):
        with pytest.raises(RuntimeError, match="unsupported"):
            size(**bad)


# ---- the plain forms --------------------------------------------------------------------------------------------------
def test_plain_tables_take_back_what_they_gave():
    t = ops.page_tables(4, 10, 20, "cpu")
    rows, new = torch.tensor([2, 0]), torch.tensor([17, 5])
    li = ref.tables_grow(t.table, t.lengths, t.free_pages, t.free_count, rows, new)
    assert li["kv_indices"] == [0, 1, 2] and li["kv_last_page_len"] == [1, 5] and li["slots"][:3] == [0, 1, 2] and li["slots"][16:18] == [16, 32]
    ref.tables_trim(t.table, t.lengths, t.free_pages, t.free_count, rows, torch.tensor([1, 9]))
    assert t.lengths.tolist() == [0, 0, 16, 0] and t.free_count.tolist() == [19] and t.free_pages[17:19].tolist() == [2, 1]


def test_plain_accept_takes_the_first_child():
    paths, following, dropped = ref.tree_accept(torch.tensor([5, 7, 7, 9, 3]), torch.tensor([-1, 0, 0, 1, 2]), torch.tensor([7, 9, 3, 4, 0]), torch.tensor([0, 5]), 9)
    assert paths == [[0, 1, 3]] and following == [4] and dropped == [2]
