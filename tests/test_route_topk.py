"""The router alone on the device (route_topk): refusals, sizes, and calls that overlap on the GPU."""
import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200._lib import MoEError


@pytest.fixture
def plane(monkeypatch):
    """A plane of the host's memory whose C calls get a null context."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    return p


@pytest.mark.parametrize("shape", [(7,), (9,), (1,), (0,), (8, 8), ()])
def test_a_bias_of_another_size_is_refused(plane, shape):
    """A shorter one would be read behind its end."""
    with pytest.raises(ValueError, match="bias is"):
        plane.route_topk(torch.zeros(3, 8), bias=torch.zeros(shape))


def test_a_bias_of_the_experts_is_taken(plane):
    for bias in (None, torch.zeros(8), torch.zeros(1, 8), torch.zeros(8, dtype=torch.float64)):
        with pytest.raises(MoEError, match="null context"):
            plane.route_topk(torch.zeros(3, 8), bias=bias)
