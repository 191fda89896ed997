"""The device-side status beside calls that run on another stream at that time."""
import pytest
import torch

from tests.fp8_util import weight

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_an_error_is_reported_once_whatever_else_reads_the_status():
    """A status read on one stream while a call on another one fails: either that read or the next one says so."""
    from npu_offload_b200 import Fp8, MoEDataPlane
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    g = gen(1)
    with MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        x = torch.randn(1, 64, generator=g, device="cuda").to(torch.bfloat16)
        gate_up, down = Fp8(*weight(g, 8, 2, 64, 64)), Fp8(*weight(g, 8, 64, 64))
        bad, w = torch.tensor([[3, 8]], dtype=torch.int32, device="cuda"), torch.ones(1, 2, device="cuda")
        here, there = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        lost = []
        for i in range(10000):
            with torch.cuda.stream(there):
                torch.cuda._sleep(200 * (i % 500))  # the error comes a little later each time
                p.experts_fp8(x, gate_up, down, bad, w)
            seen = [p.status(here), p.status(there)]
            assert set(seen) <= {MOE_OK, MOE_EINVAL}
            if seen.count(MOE_EINVAL) != 1:
                lost.append((i, seen))
        assert not lost, (len(lost), lost[:5])
        assert p.status() == MOE_OK


def test_a_wait_that_gave_up_beside_a_running_layer_leaves_its_counts_alone():
    """A product gives up (test hook) and its status is read while layer calls run on another stream: their grids count
    arrivals over all calls, and go on from where they were."""
    from npu_offload_b200 import Fp8, MoEDataPlane
    from npu_offload_b200._lib import MOE_ETIMEOUT, MOE_OK, MOE_OPT_INJECT_WAIT_TIMEOUT, MOE_OPT_WAIT_TIMEOUT_US
    H, F, E, K, T = 512, 256, 16, 4, 2
    g = gen(2)
    with MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=16) as p:
        for e in range(E):
            p.load_expert(0, e, *((torch.randn(*s, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
                                  for s in ((F, H), (F, H), (H, F))))
        xs = [torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16) for _ in range(4)]
        lgs = [torch.randn(T, E, generator=g, device="cuda") for _ in range(4)]
        rows, w = p.quantize_fp8(torch.randn(1, 1024, generator=g, device="cuda")), Fp8(*weight(g, 100, 1024))
        want = [p.forward(0, x, lg) for x, lg in zip(xs, lgs)]
        layers, products = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        assert p.status() == MOE_OK
        got = []
        for i in range(30):
            with torch.cuda.stream(layers):
                torch.cuda._sleep(1_000_000 * (i % 5))
                got += [p.forward(0, x, lg) for x, lg in zip(xs, lgs)]
            p.set_option(MOE_OPT_WAIT_TIMEOUT_US, 1000)
            p.set_option(MOE_OPT_INJECT_WAIT_TIMEOUT, 1)
            p.matmul_fp8(rows, w, stream=products)
            p.set_option(MOE_OPT_INJECT_WAIT_TIMEOUT, 0)
            p.set_option(MOE_OPT_WAIT_TIMEOUT_US, 1_000_000)
            assert p.status(products) == MOE_ETIMEOUT
        torch.cuda.synchronize()
        assert p.status() == MOE_OK
        # the plan may cut the sums elsewhere behind a running call: the same experts, not the same order of sums
        for i, y in enumerate(got):
            v = want[i % 4]
            assert float((y - v).abs().max()) <= 1e-4 * float(v.abs().max())


def test_the_status_is_not_that_of_another_runtime_call():
    """A call of the CUDA runtime that failed before, and was dealt with, is no error of the plane."""
    import ctypes

    from npu_offload_b200 import MoEDataPlane
    from npu_offload_b200._lib import MOE_OK
    with MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        assert p.status() == MOE_OK
        library = [line.split()[-1] for line in open("/proc/self/maps") if "libcudart.so" in line and "r-xp" in line]
        for path in sorted(set(library)):
            assert ctypes.CDLL(path).cudaSetDevice(10 ** 6) != 0  # no such device; leaves its code for cudaGetLastError
        assert p.status() == MOE_OK
        for path in sorted(set(library)):
            ctypes.CDLL(path).cudaGetLastError()
