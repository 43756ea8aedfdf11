"""Drafted tokens: sizes next to 32 bits, which a loop would step over, are refused before any launch."""
from ctypes import c_void_p

import pytest

import test_draft_cpu as base
from nanoflow_b200 import ops
from nanoflow_b200.ops import draft

MOST = 0x7ff00000                 # a loop's step, of all threads or of a request's share, stays below 2^20


@pytest.mark.parametrize("field", ["num_tokens", "num_indices"])
@pytest.mark.parametrize("entries", [MOST + 1, 2 ** 31 - 1])
def test_lists_of_tables_without_room_for_a_step_are_refused(field, entries):
    pointers = ("table", "lengths", "free_pages", "free_count", "ticket", "rows", "tokens", "qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len",
                "positions", "token_req", "slots")
    values = dict(requests=1, max_requests=1, max_pages=1, num_pages=1, num_indices=1, num_tokens=1)
    assert ops.lib().nfk_tables_grow(base._filled(draft.TablesParams, pointers, values, {field: entries}), c_void_p(0)) == 1


@pytest.mark.parametrize("field", ["num_tokens", "req_count"])
@pytest.mark.parametrize("entries", [MOST + 1, 2 ** 31 - 1])
def test_attention_of_more_than_a_step_leaves_room_for_is_refused(field, entries):
    pointers = ("q", "out", "kv_pool", "qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len", "tree", "workspace")
    values = dict(ld_q=64, ld_out=64, q_heads=1, kv_heads=1, head_dim=64, num_pages=4, num_tokens=3, num_indices=4, req_count=3, words=1, sm_scale=0.1,
                  workspace_bytes=1 << 40)
    assert ops.lib().nfk_attn_tree(base._filled(draft.AttnTreeParams, pointers, values, {field: entries}), c_void_p(0)) == 1


@pytest.mark.parametrize("entries", [MOST + 1, 2 ** 31 - 1])
def test_trees_of_more_than_a_step_leaves_room_for_are_refused(entries):
    masks, accept = dict(requests=1, num_tokens=1, words=1), dict(requests=1, num_tokens=1, max_path=1)
    for field in ("num_tokens", "requests", "max_path"):
        if field != "max_path":
            assert ops.lib().nfk_tree_masks(base._filled(draft.TreeMasksParams, ("parents", "qo_indptr", "mask"), masks, {field: entries}), c_void_p(0)) == 1
        pointers = ("tokens", "parents", "targets", "qo_indptr", "path", "counts", "next_tokens")
        assert ops.lib().nfk_tree_accept(base._filled(draft.TreeAcceptParams, pointers, accept, {field: entries}), c_void_p(0)) == 1


@pytest.mark.parametrize("field", ["num_qo", "num_kv", "num_last"])
def test_lists_of_requests_without_room_for_a_step_are_refused(field):
    test_lists_of_tables_without_room_for_a_step_are_refused(field, MOST + 1)


# ---- frequencies: entries of a configuration that are null, or none that a rotation has ------------------------------------------------
@pytest.mark.parametrize("scaling,more", [
    ({"rope_type": "linear", "factor": None}, {}), ({"rope_type": "dynamic", "factor": None}, {"max_position": 4096}), ({"rope_type": "llama3", "factor": None}, {}),
    ({"rope_type": "yarn", "factor": None, "original_max_position_embeddings": 4096}, {}),
    ({"rope_type": "longrope", "short_factor": None, "long_factor": [1.0] * 32}, {"max_position": 4096}),
    ({"rope_type": "longrope", "short_factor": [1.0] * 31 + [0.0], "long_factor": [1.0] * 32}, {"max_position": 4096}),
    ({"rope_type": "longrope", "short_factor": [1.0] * 32, "long_factor": [1.0] * 32, "original_max_position_embeddings": 1}, {"max_position": 4096}),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0}, {}),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 0.0}, {}), ({"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": -1}, {}),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "beta_fast": -32}, {}),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": -4096}, {}), ({"rope_type": "linear", "factor": float("nan")}, {}),
    ({"rope_type": "linear", "factor": float("inf")}, {}), ({"rope_type": "dynamic", "factor": 2.0}, {"max_position": -5})])
def test_frequencies_refuse_what_is_none(scaling, more):
    with pytest.raises(RuntimeError, match="rope_frequencies"):
        ops.rope_frequencies(64, 10000.0, scaling, device="cpu", **more)


def test_frequencies_take_null_for_what_has_a_default():
    for null, plain in (({"rope_type": None}, {}), ({"rope_type": None, "type": "linear", "factor": 2.0}, {"type": "linear", "factor": 2.0}),
                        ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": None, "high_freq_factor": None, "original_max_position_embeddings": None},
                         {"rope_type": "llama3", "factor": 8.0}),
                        ({"rope_type": "yarn", "factor": None, "original_max_position_embeddings": 1024, "attention_factor": None, "beta_fast": None, "truncate": None},
                         {"rope_type": "yarn", "original_max_position_embeddings": 1024})):
        a, b = (ops.rope_frequencies(64, 10000.0, s, max_position=4096, device="cpu") for s in (null, plain))
        assert a[0].tolist() == b[0].tolist() and a[1] == b[1]
