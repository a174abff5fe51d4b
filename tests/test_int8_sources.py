"""What the sources of the 8-bit kernels have to hold by their wording, because a run shows only what one compiler made of it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-runtime-byyourself_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name), encoding="utf-8") as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["gemm_int8.cu", "int8_rows.cu"])
def test_loads_stay_behind_the_wait_for_the_kernel_ahead(name):
    """A product may follow the kernel that quantised its weights by one launch.  A load in assembly that is not volatile, names no memory or is of memory
    that no one writes (.nc) may be moved ahead of the wait for that kernel."""
    text = source(name)
    loads = re.findall(r"asm\s*(volatile)?\s*\(([^;]*?ld\.global.*?)\)\s*;\s*(?:\n|$)", text, flags=re.S)
    assert len(loads) == text.count("ld.global")
    for volatile, body in loads:
        assert volatile and '"memory"' in body and ".nc" not in body, body
    assert "__ldg(" not in text


def test_a_block_waits_for_its_copies_before_it_goes():
    """Also where another role of the block has given up: each producer's last step is to wait until every stage has been handed back."""
    text = source("gemm_int8.cu")
    kernels = re.split(r"__global__", text)[1:]
    producers = [k for k in kernels if "tma_load_2d" in k]
    assert len(producers) == 2
    for kernel in producers:
        role = kernel[kernel.index("if (warp == 0) {"):kernel.index("else if (warp == 1) {", kernel.index("if (warp == 0) {"))]
        assert role.rindex("wait_for_stages<STAGES>(bars + STAGES * 8,") > role.rindex("tma_load_2d")
