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
