"""Sizes at the ends of what the products in 8 bits take: their plan, and what is refused before a launch."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CALLS = """
import ctypes, sys
sys.path.insert(0, {root!r})
from qwen3_b200.csrc import ops
lib = ops.load_library("gemm_int8.cu", ())
splits = ctypes.c_int(0)
for rows, channels, width in ((1, 1, 1), (64, 4096, 4096), (527, 5120, 17408), (0x7fffffff, 0x7fffffff, 131071), (0x7fffffff, 16, 1), (16, 0x7fffffff, 64), (0, 4, 4)):
    assert lib.q3_gemm_int8_plan(rows, channels, width, ctypes.byref(splits)) in (0, 1, 2)
for rows, channels in ((0x7fffffff, 16), (16, 0x7fffffff), (0x7fffffff - 255, 16)):
    for form in ("few", "mid", "pair"):
        args = ops._GEMM8_ARGS.pack(1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, 16, 16, rows, channels, 16, 0, 0, 0)
        code = getattr(lib, "q3_gemm_int8_" + form)(args)
        assert code == 10002, (form, rows, channels, code)
print("done")
"""


def test_plans_and_sizes_without_a_device():
    """In a process of its own: without a device, whose SMs the plan counts, it once divided by zero.  Sizes that 32 bits do not count to are refused before a launch."""
    done = subprocess.run([sys.executable, "-c", CALLS.format(root=ROOT)], capture_output=True, text=True, timeout=600, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert done.returncode == 0 and "done" in done.stdout, (done.returncode, done.stderr[-2000:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels,width", [(17_000_000, 64, 8192), (16_777_000, 128, 4096), (20_000_000, 16, 4096), (1, 25600, 131071), (64, 64, 64),
                                                 (0x7ffffeff, 16, 16), (8000, 24576, 4096)])
def test_plans_can_be_launched(rows, channels, width):
    """A grid takes 65,535 tiles of tokens along an axis; `splits` are K ranges of a cluster, or a tile's tokens."""
    from qwen3_b200.csrc import ops
    form, splits = ops.int8_plan(rows, channels, width)
    assert form in ("few", "mid", "pair")
    if form == "mid":
        assert -(-rows // 256) <= 65535 and 1 <= splits <= 8
    elif form == "pair":
        assert splits % 32 == 0 and 32 <= splits <= 256 and -(-rows // splits) * -(-channels // 256) <= 0x3FFFFFFF


@pytest.mark.gpu
@pytest.mark.parametrize("rows,channels,width,form", [(1, 4096, 4096, "few"), (8, 4096, 12288, "few"), (8, 24576, 4096, "few"), (64, 6144, 4096, "mid"),
                                                      (1024, 4096, 4096, "pair"), (2048, 24576, 4096, "pair"), (8000, 4096, 12288, "pair")])
def test_forms_of_sizes_where_the_others_are_far_behind(rows, channels, width, form):
    """A token alone streams W; some dozen share it in tensor memory, K split over a cluster; a thousand and more fill the pairs of SMs."""
    from qwen3_b200.csrc import ops
    assert ops.int8_plan(rows, channels, width)[0] == form
