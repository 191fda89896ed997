"""What the adapters' call refuses and takes, without a GPU."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200 import _lib
from npu_offload_b200._lib import MoEError

BF = torch.bfloat16


@pytest.fixture
def plane(monkeypatch):
    """A plane of the host's memory whose C calls get a null context."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    return p


def args(**kw):
    a = dict(base=torch.zeros(3, 20), x=torch.zeros(3, 32, dtype=BF), a=torch.zeros(4, 8, 32, dtype=BF), b=torch.zeros(4, 20, 8, dtype=BF),
             ids=torch.zeros(3, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,needle", [
    (dict(base=torch.zeros(3, 20, dtype=torch.float16)), "float16"),
    (dict(base=torch.zeros(3, 21)), "base is"),
    (dict(base=torch.zeros(2, 20)), "base is"),
    (dict(base=None), "tensor on"),
    (dict(x=torch.zeros(3, 32)), "float32"),
    (dict(x=torch.zeros(3, 40, dtype=BF)), "a is"),
    (dict(x=torch.zeros(1, 3, 32, dtype=BF)), "dimensions"),
    (dict(a=torch.zeros(4, 8, 32)), "float32"),
    (dict(a=torch.zeros(8, 32, dtype=BF)), "dimensions"),
    (dict(a=torch.zeros(4, 32, 8, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(a=torch.zeros(4 * 8 * 32 + 1, dtype=BF)[1:].view(4, 8, 32)), "aligned"),
    (dict(b=torch.zeros(3, 20, 8, dtype=BF)), "b is"),
    (dict(b=torch.zeros(4, 20, 16, dtype=BF)), "b is"),
    (dict(b=torch.zeros(4, 8, 20, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(ids=torch.zeros(3, dtype=torch.int64)), "int64"),
    (dict(ids=torch.zeros(2, dtype=torch.int32)), "ids has"),
    (dict(scale=torch.ones(3)), "scale has"),
    (dict(scale=torch.ones(4, dtype=torch.float64)), "float64"),
    (dict(out=torch.zeros(3, 19)), "out must be"),
    (dict(out=torch.zeros(3, 20, dtype=BF)), "out is"),
    (dict(x=torch.zeros(3, 32, dtype=BF, requires_grad=True)), "autograd"),
    (dict(a=torch.zeros(4, 8, 32, dtype=BF, requires_grad=True)), "autograd"),
    (dict(b=torch.zeros(4, 20, 8, dtype=BF, requires_grad=True)), "autograd"),
    (dict(base=torch.zeros(3, 20, requires_grad=True)), "autograd"),
    (dict(scale=torch.ones(4, requires_grad=True)), "autograd"),
])
def test_add_lora_refuses(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.add_lora(**args(**kw))


def test_add_lora_takes_what_is_documented(plane):
    base = torch.zeros(3, 20)
    for kw in (dict(), dict(base=base, out=base), dict(base=base.to(BF)), dict(scale=torch.ones(4)), dict(x=torch.zeros(32, 3, dtype=BF).T),
               dict(base=torch.zeros(0, 20), x=torch.zeros(0, 32, dtype=BF), ids=torch.zeros(0, dtype=torch.int32))):
        with pytest.raises(MoEError, match="null context"):
            plane.add_lora(**args(**kw))
    with torch.no_grad(), pytest.raises(MoEError, match="null context"):
        plane.add_lora(**args(a=torch.zeros(4, 8, 32, dtype=BF, requires_grad=True)))


def test_a_stream_of_another_device_is_refused(plane, monkeypatch):
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    plane.device = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        plane.add_lora(**args(), stream=SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=5))


def test_c_entry_points_report_a_null_context():
    L = nob.lib()
    assert L.moe_add_lora_workspace(None, 1, 8, 1) == -1
    assert L.moe_add_lora(None, 1, 8, 8, 8, 1, None, None, None, None, None, None, None, 0, None, 0, 0, None) == _lib.MOE_EINVAL
