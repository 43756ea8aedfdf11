"""The shared prefix's states: a CTA that gives up (a wait that ran out) leaves one for each of its parts all the same, NaN, so that no
state of an earlier call is joined in its place."""
import subprocess

import pytest

from nanoflow_b200.ops import build


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    build.build_kernels()
    out = tmp_path_factory.mktemp("pieces") / "pieces"
    source = build.ROOT / "tests" / "cache_q8_pieces.cu"
    build._run([build.NVCC, *build.ARCH_FLAGS, "-std=c++17", "--expt-relaxed-constexpr", "-I", build.KERNEL_DIR, source, "-o", out, "-L", build.KERNEL_LIB.parent,
                "-l:libnanoflow_kernels.so", "-Xlinker", f"-rpath={build.KERNEL_LIB.parent}"], False)
    return out


@pytest.mark.parametrize("requests,heads,kv_heads,prefix,ctas", [
    (1, 8, 2, 1, 0), (1, 8, 2, 65, 0), (5, 8, 2, 5000, 3), (70, 16, 4, 3333, 7), (70, 16, 4, 3333, 0), (2, 3, 1, 9001, 40), (9, 32, 8, 700, 5),
    (256, 32, 8, 8192, 0), (64, 64, 8, 32768, 0), (16, 32, 8, 1999, 0), (8, 16, 1, 30000, 0), (400, 28, 4, 777, 0), (1000, 9, 3, 64, 1)])
def test_every_state_that_is_read_is_written(program, requests, heads, kv_heads, prefix, ctas):
    done = subprocess.run([str(program), *map(str, (requests, heads, kv_heads, prefix, ctas))], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_the_kernel_spoils_what_it_does_not_compute():
    text = (build.KERNEL_DIR / "attn_prefix_q8.cu").read_text()
    softmax = text[text.index("softmax (a thread per query row)"):]
    assert "if (!ok) now.rest(spoil);" in softmax and softmax.count("ok = false; break;") == softmax.count("fail(NF_ST_")
    assert "all.rest(spoil);" in text[:text.index("mbar_init")]


def test_products_in_flight_end_before_their_memory_is_given_back():
    text = (build.KERNEL_DIR / "attn_prefix_q8.cu").read_text()
    products = text[text.index("products (the warp walks"):text.index("softmax (a thread per query row)")]
    assert products.count("ok = false; break;") == products.count("fail(NF_ST_")
    end = products[products.rindex("if (!ok) {"):]
    assert end.index("umma_commit(&bars[C::LAST])") < end.index("mbar_wait(&bars[C::LAST], 0)")
    assert text.index("mbar_wait(&bars[C::LAST], 0)") < text.index("tmem_dealloc(")
