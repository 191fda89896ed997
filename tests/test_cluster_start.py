"""Kernels that reach into another CTA's shared memory do so only once the whole cluster is known to run."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu_offload_b200", "csrc")
REMOTE = re.compile(r"map_shared_rank\s*\(|cluster_map\s*\(")
BARRIER = re.compile(r"\bcl\.sync\s*\(\)|cluster_sync_all\s*\(\)")


def kernels():
    """(file, name, body) of every kernel whose body reaches into a cluster's shared memory."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__", text):
            start = text.index("{", m.end())
            depth, end = 1, start + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            body = text[start:end]
            if REMOTE.search(body):
                name = re.search(r"(\w+)\s*\([^()]*(\([^()]*\)[^()]*)*\)\s*$", text[m.end():start]).group(1)
                found.append((os.path.basename(path), name, body))
    return found


def test_the_kernels_are_found():
    assert {"balance_sum_kernel", "f8_plan_kernel", "f8_few_kernel"} <= {k[1] for k in kernels()}


@pytest.mark.parametrize("file,name,body", kernels(), ids=[k[1] for k in kernels()])
def test_the_cluster_meets_before_the_first_remote_access(file, name, body):
    barrier = BARRIER.search(body)
    assert barrier and barrier.start() < REMOTE.search(body).start(), f"{file}: {name}"


@pytest.mark.gpu
def test_lone_calls_of_one_to_many_clusters():
    """The sums of one cluster, of all that fit at once and of more, each call on a GPU that has nothing else to run."""
    import torch

    from npu_offload_b200 import MoEDataPlane
    from tests.fp8_util import EPS, balance64
    g = torch.Generator(device="cuda").manual_seed(2)
    with MoEDataPlane(64, 64, 64, 4, n_layers=1, max_tokens=16) as p:
        logits = torch.randn(600, 64, generator=g, device="cuda")
        idx = logits.topk(4, -1)[1].int()
        for B in (1, 2, 18, 19, 300):
            off = torch.linspace(0, 600, B + 1, device="cuda").int()
            want, counts, _ = balance64(logits, idx, off, None, "softmax")
            for _ in range(20):
                loss, st = p.balance_loss(logits, idx, offsets=off)
                torch.cuda.synchronize()
                assert torch.equal(st.counts, counts)
                # a score is off by the logits' span, exp, the sum and the quotient, in half steps
                assert abs(float(loss) - float(want)) <= (float(logits.max() - logits.min()) + 56) * EPS * float(want)
        assert p.status() == 0
