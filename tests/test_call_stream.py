"""The stream= argument of the calls that allocate through torch: one of the plane's device, or refused."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import npu_offload_b200 as nob

F8 = torch.float8_e4m3fn


@pytest.fixture
def plane(monkeypatch):
    """A plane of cuda:0 without a context, on a host without a GPU."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cuda", 0)
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    return p


def calls(p, stream):
    x, lg = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 8)
    idx = torch.zeros(3, 2, dtype=torch.int32)
    q = nob.Fp8(torch.zeros(3, 256).to(F8), torch.ones(3, 2))
    st = nob.BalanceStats(torch.zeros(1, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), None, None)
    return {
        "quantize_fp8": lambda: p.quantize_fp8(x, stream=stream),
        "matmul_fp8": lambda: p.matmul_fp8(q, q, stream=stream),
        "experts_fp8": lambda: p.experts_fp8(x, q, q, idx, torch.zeros(3, 2), stream=stream),
        "route_topk": lambda: p.route_topk(lg, stream=stream),
        "balance_loss": lambda: p.balance_loss(lg, idx, stream=stream),
        "balance_loss_backward": lambda: p.balance_loss_backward(lg, st, stream=stream),
    }


NAMES = list(calls(None, None))


@pytest.mark.parametrize("name", NAMES)
def test_a_stream_of_another_device_is_refused(plane, name):
    """It was entered, and the call then ran on the plane's own current stream, out of the caller's order."""
    other = SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=5)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        calls(plane, other)[name]()


@pytest.mark.parametrize("name", NAMES)
def test_a_stream_of_the_device_is_entered(plane, name):
    own = SimpleNamespace(device=torch.device("cuda", 0), cuda_stream=5)
    with pytest.raises(Exception) as e:  # what the call says of tensors of the host
        calls(plane, own)[name]()
    assert "stream is on" not in str(e.value)
