"""The norm, grouped routing and adapter kernels start before the end of the ones before them.  Read from their source: each touches
memory of the call's arguments behind its wait alone, but for lora_out_kernel, whose reads ahead of it go past L1; and no kernel
calls, directly or through the headers, what loads non-coherently."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu_offload_b200", "csrc")
FILES = ["norm.cu", "norm_backward.cu", "route_groups.cu", "lora.cu", "lora_many.cu"]
NON_COHERENT = r"\b__ldg\b|\.nc\b|\b__restrict__\b"


def text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def block(s, at):
    """What stands between the braces of which the first is the next from `at` on."""
    start = s.index("{", at)
    depth = 0
    for i in range(start, len(s)):
        depth += {"{": 1, "}": -1}.get(s[i], 0)
        if depth == 0:
            return s[start + 1:i]
    raise AssertionError("a brace is not closed")


def kernels(name):
    """{kernel: (parameters, body)} of a file."""
    s, out = text(name), {}
    for m in re.finditer(r"__global__\b", s):
        head = s[m.end():s.index("{", m.end())]
        k = re.search(r"(\w+)\s*\(([^()]*)\)\s*$", head)
        out[k[1]] = k[2], block(s, m.end())
    return out


def pointers():
    """Names of the argument structs' fields that point to memory of a call."""
    names = set()
    for f in ("norm.h", "route_groups.h", "lora.h", "lora_many.cu"):
        for m in re.finditer(r"struct (\w*(?:Args|Ws)) ", text(f)):
            names |= set(re.findall(r"\*\s*(\w+)\s*;", block(text(f), m.end())))
    return names


def parameters(params):
    return set(re.findall(r"\*\s*(\w+)", params))


def test_the_files_are_all_that_launch_this_way():
    found = [f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and re.search(r"\bconst Launch \w+\{", text(f))]
    assert sorted(found) == sorted(FILES)
    assert {"x", "base", "ids", "err", "logits", "dw", "rstd", "order", "low", "tiles"} <= pointers()
    for f in FILES:
        assert kernels(f), f
    assert set(kernels("lora_many.cu")) == {"lora_plan_kernel", "lora_low_kernel", "lora_out_kernel"}
    assert {"route_groups_kernel", "route_octet_kernel", "route_backward_kernel", "route_dense_kernel"} == set(kernels("route_groups.cu"))


def ahead(body):
    assert "griddep_wait()" in body
    return body[:body.index("griddep_wait()")]


@pytest.mark.parametrize("name", FILES)
def test_nothing_of_the_arguments_is_touched_ahead_of_the_wait(name):
    for kernel, (params, body) in kernels(name).items():
        if kernel == "lora_out_kernel":
            continue
        before = ahead(body)
        used = {m[1] for m in re.finditer(r"\b(?:a|ws|p)(?:\.|->)(\w+)", before)} & pointers()
        assert not used, (kernel, used)
        assert not [p for p in parameters(params) if re.search(rf"\b{p}\b", before)], kernel


def test_what_the_last_adapter_kernel_reads_ahead_goes_past_l1():
    before = ahead(kernels("lora_many.cu")["lora_out_kernel"][1])
    assert set(re.findall(r"\bws\.(\w+)", before)) == {"n_tiles", "order", "tiles"}  # of the kernel before the one before
    assert set(re.findall(r"\ba\.(\w+)", before)) & pointers() == {"base", "b"}
    assert not re.search(r"\ba\.out\b(?!_)", before)
    # memory is named as the argument of these alone
    for at in re.finditer(r"\bws\.(n_tiles|tiles)|\border \+", before):
        line = before[before.rindex(";", 0, at.start()):before.index(";", at.end())]
        assert "__ldcg(" in line or re.search(r"const int(32_t)?\* order =", line), line
    for at in re.finditer(r"\ba\.base\b|\ba\.b\b", before):
        line = before[before.rindex(";", 0, at.start()):before.index(";", at.end())]
        assert "cp_async16_or_zero(" in line or "const uint16_t* B =" in line, line
    assert not re.search(r"\b(B|order|low|tiles|base)\s*\[|\*\s*(reinterpret_cast|static_cast)|=\s*\*", before)
    assert "cp.async.cg.shared.global" in block(text("lora_many.cu"), text("lora_many.cu").index("cp_async16_or_zero("))


def includes(name, seen=None):
    seen = set() if seen is None else seen
    for f in re.findall(r'#include "([^"]+)"', text(name)):
        if f not in seen and os.path.exists(os.path.join(CSRC, f)):
            seen.add(f)
            includes(f, seen)
    return seen


@pytest.mark.parametrize("name", FILES)
def test_nothing_loads_non_coherently(name):
    assert not re.search(NON_COHERENT, text(name))
    functions = {}
    for f in includes(name):
        s = text(f)
        for m in re.finditer(r"\b(\w+)\s*\([^;{}()]*(?:\([^()]*\)[^;{}()]*)*\)\s*\{", s):
            functions[m[1]] = functions.get(m[1], "") + block(s, m.start())
    bad = {f for f, body in functions.items() if re.search(NON_COHERENT, body)}
    assert name != "norm.cu" or "ldg_stream" in bad  # (it is found where it is)
    while True:
        more = {f for f, body in functions.items() if f not in bad and any(re.search(rf"\b{b}\s*\(", body) for b in bad)}
        if not more:
            break
        bad |= more
    used = [b for b in bad if re.search(rf"\b{b}\s*[(<]", text(name))]
    assert not used, used


@pytest.mark.parametrize("name", FILES)
def test_only_kernels_with_one_behind_them_let_it_start(name):
    for kernel, (_, body) in kernels(name).items():
        lets = "griddep_launch_dependents()" in body
        assert lets == (kernel in ("lora_plan_kernel", "lora_low_kernel", "norm_backward_kernel")), kernel
        assert not lets or body.index("griddep_wait()") < body.index("griddep_launch_dependents()")
