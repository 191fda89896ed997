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


def test_launches_of_several_threads_are_all_counted():
    """The calls that may overlap on one context keep the launch count, each thread on its own stream."""
    import ctypes
    import threading

    import torch

    from npu_offload_b200 import MoEDataPlane, lib
    with MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        logits = torch.randn(4, 8, device="cuda")
        outs = [(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")) for _ in range(8)]
        streams = [torch.cuda.Stream() for _ in outs]
        want = p.route_topk(logits)
        torch.cuda.synchronize()
        before, n, bad = p.launch_count, 3000, []

        def call(i):
            a = [ctypes.c_void_p(t.data_ptr()) for t in (logits, *outs[i])]
            for _ in range(n):
                if lib().moe_route_topk(p._h, 4, a[0], None, a[1], a[2], 0, ctypes.c_void_p(streams[i].cuda_stream)):
                    bad.append(i)

        threads = [threading.Thread(target=call, args=(i,)) for i in range(len(outs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not bad and p.launch_count - before == n * len(outs)
        assert all(torch.equal(o[0], want[0]) and torch.equal(o[1], want[1]) for o in outs)
        assert p.status() == 0
