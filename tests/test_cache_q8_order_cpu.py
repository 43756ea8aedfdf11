"""Kernels of attention over the 8-bit cache read lists and queries before their wait for the kernel in front of them: what makes that
sound stands in the sources (a fence in front of the launch, loads by way of L2) and cannot be seen from results."""
import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "nanoflow_b200" / "csrc" / "kernels"


def _kernels(name):
    """{name: body} of the file's kernels, without comments."""
    text = re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())
    found = {}
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\([^{]*?\)\s*)?(\w+)\(", text):
        at = text.index("{", m.end())
        depth, i = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        found[m.group(1)] = text[at:i]
    return found


def test_what_is_read_early_is_read_through_l2():
    """Lists and queries are reached by Early alone where the kernel has not waited, and Early goes to L2 there."""
    kernels = _kernels("attn_decode_q8.cu")
    assert {"attn_decode_q8_kernel", "attn_join_parts_q8_kernel", "attn_join_rows_q8_kernel"} <= set(kernels)
    for name, body in kernels.items():
        for use in re.finditer(r"\bp\.(q|kv_indptr|kv_indices|qo_indptr|kv_last_page_len)\b", body):
            assert re.search(r"\bEarly<\w+(, SHARED)?> [^;]*$", body[:use.start()]), (name, use.group(0))
    assert re.search(r"constexpr bool SHARED = MODE == SHARED_PREFIX;", kernels["attn_decode_q8_kernel"])
    assert "if (!SHARED) await_previous();" in kernels["attn_decode_q8_kernel"]
    common = (KERNELS / "common.cuh").read_text()
    assert re.search(r"template <class T, bool ON = true>\s*struct Early \{[^}]*if constexpr \(ON\) return __ldcg\(at \+ i\);", common)
    assert "cp.async.cg" in (KERNELS / "attn_mma.cuh").read_text()


def test_kernels_that_others_read_behind_fence_in_front_of_their_launch():
    prefix = _kernels("attn_prefix_q8.cu")["attn_prefix_q8_kernel"]
    assert prefix.index("await_previous();") < prefix.index("let_next_read();") and "let_next_start" not in prefix
    decode = _kernels("attn_decode_q8.cu")["attn_decode_q8_kernel"]
    assert re.search(r"if \(!SHARED\) await_previous\(\);\s*if \(MODE != PLAIN\) let_next_start\(\);\s*else if \([^\n]*\) let_next_read\(\);", decode)
    common = (KERNELS / "common.cuh").read_text()
    assert re.search(r"void let_next_read\(\) \{\s*if \(elect_one\(\)\) \{[^\n]*\n\s*__threadfence\(\);\s*let_next_start\(\);", common)


def test_one_block_of_a_grid_that_starts_without_a_wait_ends_behind_it():
    decode = _kernels("attn_decode_q8.cu")["attn_decode_q8_kernel"]
    assert "if (SHARED && blockIdx.x == gridDim.x - 1) await_previous();" in decode
