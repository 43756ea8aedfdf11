"""Calls of the 8-bit cache refuse tensors that lie over one another where one of them is written; nothing is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import test_cache_q8_gpu as base


def _over(t, dtype, n, first=0):
    """n elements of `dtype` on t's memory, from its element `first` (of that type) on."""
    return t.view(-1).view(torch.uint8).view(dtype)[first:first + n]


CASES = [
    ("append", "q_out", lambda a: _over(a["kv_pool"], torch.bfloat16, 512).view(2, 256)),
    ("append", "q_out", lambda a: _over(a["kv_pool"], torch.bfloat16, 512, 4096).view(2, 256)),
    ("append", "kv_scale", lambda a: _over(a["kv_pool"], torch.float32, 384).view(6, 2, 2, 16)),
    ("append", "qkv", lambda a: _over(a["kv_pool"], torch.bfloat16, 1024).view(2, 512)),
    ("append", "positions", lambda a: _over(a["kv_scale"], torch.int32, 2, 8)),
    ("append", "token_req", lambda a: _over(a["q_out"], torch.int32, 2, 254)),
    ("append", "kv_indptr", lambda a: _over(a["kv_scale"], torch.int32, 3)),
    ("append", "kv_indices", lambda a: _over(a["kv_pool"], torch.int32, 4, 64)),
    ("append", "inv_freq", lambda a: _over(a["kv_scale"], torch.float32, 32, 64)),
    ("append", "q_norm", lambda a: _over(a["q_out"], torch.bfloat16, 64)),
    ("append", "k_norm", lambda a: _over(a["kv_pool"], torch.bfloat16, 64)),
    ("append", "cos_sin", lambda a: _over(a["kv_scale"], torch.float32, 128)),
    ("append", "status", lambda a: a["positions"]),
    ("append", "status", lambda a: _over(a["kv_scale"], torch.int32, 1, 3)),
    ("read", "out", lambda a: _over(a["kv_pool"], torch.bfloat16, 8192)[:8192].view(2, 2, 2, 16, 64)[:1]),
    ("read", "page_ids", lambda a: _over(a["out"], torch.int32, 2, 77)),
    ("read", "status", lambda a: a["page_ids"]),
    ("decode", "out", lambda a: _over(a["kv_pool"], torch.bfloat16, 512).view(2, 256)),
    ("decode", "out", lambda a: _over(a["kv_scale"], torch.bfloat16, 512).view(2, 256)),
    ("decode", "out", lambda a: _over(a["workspace"], torch.bfloat16, 512).view(2, 256)),
    ("decode", "workspace", lambda a: None),      # (a pool within the workspace: below)
    ("decode", "q", lambda a: _over(a["workspace"], torch.bfloat16, 512, 512).view(2, 256)),
    ("decode", "kv_scale", lambda a: _over(a["workspace"], torch.float32, 384).view(6, 2, 2, 16)),
    ("decode", "qo_indptr", lambda a: _over(a["workspace"], torch.int32, 2)),
    ("decode", "kv_indptr", lambda a: _over(a["out"], torch.int32, 3)),
    ("decode", "kv_indices", lambda a: _over(a["workspace"], torch.int32, 5, 64)),
    ("decode", "kv_last_page_len", lambda a: _over(a["out"], torch.int32, 2, 254)),
    ("decode", "prefix_pages", lambda a: _over(a["workspace"], torch.int32, 2, 1000)),
    ("decode", "status", lambda a: a["kv_last_page_len"]),
    ("decode", "status", lambda a: _over(a["workspace"], torch.int32, 1)),
]


@pytest.mark.parametrize("op,name,make", CASES, ids=["%s-%s-%d" % (c[0], c[1], i) for i, c in enumerate(CASES)])
def test_overlaps_are_refused(op, name, make):
    call, args, written = base._refusal_arguments()[op]
    if op == "append":
        args["cos_sin"] = None
    if name == "workspace":
        args["kv_pool"] = args["workspace"][4096:4096 + args["kv_pool"].numel()].view(torch.int8).view(args["kv_pool"].shape)
    else:
        args[name] = make(args)
    if op == "read" and name == "out":
        args["page_ids"] = args["page_ids"][:1]
    kept = [args[k].view(-1).view(torch.uint8) for k in (written, "kv_scale", "kv_pool")]      # (bytes: some of them are NaN)
    before = [t.clone() for t in kept]
    with pytest.raises(RuntimeError, match="overlap"):
        call(**args)
    torch.cuda.synchronize()
    assert all(torch.equal(t, b) for t, b in zip(kept, before))


@pytest.mark.parametrize("op", ["append", "read", "decode"])
def test_neighbours_are_not_overlaps(op):
    """All of a call's tensors one behind the other in one buffer."""
    call, args, written = base._refusal_arguments()[op]
    tensors = {k: v for k, v in args.items() if isinstance(v, torch.Tensor)}
    place, at = {}, 0
    for k, v in tensors.items():
        place[k] = at
        at += -(-v.numel() * v.element_size() // 256) * 256
    buffer = torch.zeros(at, dtype=torch.uint8, device="cuda")
    moved = {k: buffer[place[k]:place[k] + v.numel() * v.element_size()].view(v.dtype).view(v.shape) for k, v in tensors.items()}
    for k, v in tensors.items():
        moved[k].copy_(v)
    call(**args)
    call(**{**args, **moved})
    assert torch.equal(moved[written], args[written]) and torch.equal(moved["kv_pool"], args["kv_pool"])
