"""What the int8 product may read while the kernel in front of it runs (no GPU: whether a read is ordered cannot be seen in its
result). The weights of a call may have been written by any earlier kernel of the stream, the one before last included."""

import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "mylocal_llm_b200" / "csrc" / "int8_gemm.cu").read_text()


def kernel(name):
    """The text of a kernel's body."""
    at = SOURCE.index("{", re.search(r"__global__[^;{]*?\b%s\(" % name, SOURCE).end())
    depth, end = 1, at
    while depth:
        end += 1
        depth += {"{": 1, "}": -1}.get(SOURCE[end], 0)
    return re.sub(r"//[^\n]*", "", SOURCE[at:end])


def test_the_quantiser_lets_the_product_start_when_what_precedes_it_is_complete():
    body = kernel("int8_quantize_kernel")
    assert 0 <= body.index("chain_wait()") < body.index("chain_trigger()")


def test_the_tile_kernel_reads_weights_early_only_behind_the_quantiser():
    body = kernel("int8_tile_kernel")
    wait = body.index("if (!a.early) chain_wait();")
    assert wait < body.index("a.w_scales") and wait < body.index("&wmap")
    assert re.search(r"b200q_int8_gemm\([^{]*\{\s*return checked_gemm\([^;]*, false, stream\);", SOURCE)
    assert re.search(r"b200q_int8_gemm_behind_quantize\([^{]*\{\s*return checked_gemm\([^;]*, true, stream\);", SOURCE)


def test_the_pair_kernel_waits_before_every_read():
    body = kernel("int8_pair_kernel")
    first = body.index("chain_wait()")
    assert first < body.index("&xmap") and first < body.index("&wmap") and first < body.index("a.w_scales")
