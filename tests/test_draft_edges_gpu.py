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
