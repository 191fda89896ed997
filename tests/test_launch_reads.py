"""Kernels that start before the end of the ones before them read what those write with coherent loads only: the
non-coherent ones (__ldg, ld.global.nc, and what the compiler makes of const __restrict__ pointers) are for memory that
does not change while the kernel runs, and may be moved ahead of the kernel's wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu_offload_b200", "csrc")
FILES = ["fp8_quant.cu", "fp8_gemm.cu", "fp8_tc.cuh", "balance.cu"]


@pytest.mark.parametrize("name", FILES)
def test_no_load_that_may_pass_the_wait(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    assert "griddep_wait" in text
    for word in (r"\b__ldg\b", r"\bldg_stream\b", r"\b__restrict__\b", r"\.nc\b"):
        assert not re.search(word, text), word


def test_the_list_is_of_all_files_that_launch_ahead():
    found = [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and "launch_after(" in open(os.path.join(CSRC, f)).read()]
    assert set(found) - {"launch.cuh"} <= set(FILES)
