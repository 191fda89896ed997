"""Kernels that Launch::run starts wait first and read with coherent loads only, as those that launch_after starts do."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu_offload_b200", "csrc")


def text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and "const Launch " in open(os.path.join(CSRC, f)).read())


def test_there_are_such_files():
    assert {"norm.cu", "norm_backward.cu"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_no_load_that_may_pass_the_wait(name):
    for word in (r"\b__ldg\b", r"\bldg_stream\b", r"\b__restrict__\b", r"\.nc\b"):
        assert not re.search(word, text(name)), word


@pytest.mark.parametrize("name", FILES)
def test_every_kernel_waits_and_the_last_of_a_call_lets_nothing_start(name):
    bodies = text(name).split("__global__")[1:]
    assert bodies and all("griddep_wait()" in b for b in bodies)
    for b in bodies:
        if "griddep_launch_dependents" in b:
            assert b.index("griddep_wait()") < b.index("griddep_launch_dependents")
            assert re.search(r"\b(lora_plan_kernel|lora_low_kernel|norm_backward_kernel)\s*\(", b)


def test_what_they_include():
    for name in ("norm.cuh",):
        for word in (r"\b__ldg\b", r"\bldg_stream\b", r"\b__restrict__\b", r"\.nc\b"):
            assert not re.search(word, text(name)), word
