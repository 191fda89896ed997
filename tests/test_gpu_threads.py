"""Calls of several host threads through the C entry points (ctypes lets go of the interpreter's lock meanwhile)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The first product of a process, made by `n` threads at once, each with a context of its own.
FIRST = """
import ctypes, sys, threading
import torch
from npu_offload_b200 import MoEDataPlane, lib
from npu_offload_b200._lib import last_error
n = int(sys.argv[1])
planes = [MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) for _ in range(n)]
x, s = torch.zeros(32, 64, dtype=torch.uint8, device="cuda"), torch.ones(32, 1, device="cuda")
outs = [torch.ones(32, 32, device="cuda") for _ in planes]
torch.cuda.synchronize()
vp = lambda t: ctypes.c_void_p(t.data_ptr())
gate, said = threading.Barrier(n), ["not called"] * n

def call(i):
    gate.wait()
    status = lib().moe_matmul_fp8(planes[i]._h, 32, 32, 64, vp(x), vp(s), vp(x), vp(s), vp(outs[i]), 1, 0x4, None)
    said[i] = last_error() if status else ""

threads = [threading.Thread(target=call, args=(i,)) for i in range(n)]
[t.start() for t in threads]
[t.join() for t in threads]
assert said == [""] * n, said
assert all(bool((o == 0).all()) for o in outs)
"""


def run(code, *args):
    r = subprocess.run([sys.executable, "-c", code, *args], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_a_product_is_a_threads_first_call():
    """A thread that made no CUDA call yet."""
    run(FIRST, "1")


def test_the_first_product_of_a_process_by_several_threads():
    """Contexts are independent: the look-up of the tensor-map encoder, common to them, is one thread's alone."""
    for _ in range(2):
        run(FIRST, "12")
