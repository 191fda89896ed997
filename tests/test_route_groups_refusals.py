"""What routing in groups and the weights' gradient refuse and take, without a GPU; the definitions against differences."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200 import _lib
from npu_offload_b200._lib import MoEError
from tests.route_util import backward64, choose, weights64


@pytest.fixture
def plane(monkeypatch):
    """A plane of the host's memory whose C calls get a null context."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    return p


def reaches_the_library(call):
    with pytest.raises(MoEError, match="null context"):
        call()


LG, IDX, DW = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)


@pytest.mark.parametrize("kw,needle", [
    (dict(logits=torch.zeros(3, 7)), "8 experts"),
    (dict(logits=torch.zeros(8)), "dimensions"),
    (dict(logits=torch.zeros(3, 8, dtype=torch.bfloat16)), "bfloat16"),
    (dict(logits=None), "tensor on"),
    (dict(logits=torch.zeros(3, 8, requires_grad=True)), "autograd"),
    (dict(bias=torch.zeros(7)), "bias is"),
    (dict(bias=torch.zeros(1, 8)), "dimensions"),
    (dict(bias=torch.zeros(8, dtype=torch.float64)), "float64"),
    (dict(groups=1 << 40), "out of range"),
    (dict(top_groups=-(1 << 40)), "out of range"),
])
def test_route_groups_refuses(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.route_groups(**{**dict(logits=LG, groups=4, top_groups=2), **kw})


def test_route_groups_takes_what_is_documented(plane):
    for kw in (dict(), dict(bias=torch.zeros(8)), dict(bias=torch.zeros(8, requires_grad=True)), dict(logits=torch.zeros(8, 3).T),
               dict(logits=torch.zeros(0, 8)), dict(renormalize=False, scale=2.5)):
        reaches_the_library(lambda: plane.route_groups(**{**dict(logits=LG, groups=4, top_groups=2), **kw}))


@pytest.mark.parametrize("kw,needle", [
    (dict(logits=torch.zeros(3, 9)), "8 experts"),
    (dict(idx=torch.zeros(3, 3, dtype=torch.int32)), "must be"),
    (dict(idx=torch.zeros(3, 2, dtype=torch.int64)), "int64"),
    (dict(dw=torch.zeros(2, 2)), "must be"),
    (dict(dw=torch.zeros(3, 2, dtype=torch.float64)), "float64"),
    (dict(dw=torch.zeros(3, 2, requires_grad=True)), "autograd"),
    (dict(logits=torch.zeros(3, 8, requires_grad=True)), "autograd"),
    (dict(accumulate=True), "accumulate"),
    (dict(out=torch.zeros(3, 7)), "out must be"),
    (dict(out=torch.zeros(8, 3).T), "out must be"),
    (dict(out=torch.zeros(3, 8, dtype=torch.bfloat16)), "out must be"),
])
def test_backward_refuses(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.route_backward(**{**dict(logits=LG, idx=IDX, dw=DW), **kw})


def test_backward_takes_what_is_documented(plane):
    for kw in (dict(), dict(out=torch.zeros(3, 8)), dict(out=torch.zeros(3, 8), accumulate=True), dict(renormalize=False, scale=0.0)):
        reaches_the_library(lambda: plane.route_backward(**{**dict(logits=LG, idx=IDX, dw=DW), **kw}))


def test_a_stream_of_another_device_is_refused(plane, monkeypatch):
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    plane.device = torch.device("cuda", 0)
    other = SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=5)
    for call in (lambda: plane.route_groups(LG, 4, 2, stream=other), lambda: plane.route_backward(LG, IDX, DW, stream=other)):
        with pytest.raises(ValueError, match="stream is on cuda:1"):
            call()


def test_c_entry_points_report_a_null_context():
    L = nob.lib()
    assert L.moe_route_groups(None, 1, None, None, 1, 1, 1, 1.0, None, None, 0, None) == _lib.MOE_EINVAL
    assert L.moe_route_backward(None, 1, None, None, None, 1, 1.0, None, 0, None) == _lib.MOE_EINVAL


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_the_gradient_agrees_with_differences(scoring, renormalize):
    g = torch.Generator().manual_seed(2)
    l, dw = torch.randn(4, 6, generator=g, dtype=torch.float64), torch.randn(4, 3, generator=g, dtype=torch.float64)
    idx = l.topk(3, -1)[1].int()
    want, _ = backward64(l, idx, dw, scoring, renormalize, 2.5)
    f = lambda x: float((weights64(x, idx, scoring, renormalize, 2.5) * dw).sum())  # noqa: E731
    for i in range(l.numel()):
        d = torch.zeros_like(l)
        d.view(-1)[i] = 1e-6
        assert abs((f(l + d) - f(l - d)) / 2e-6 - float(want.view(-1)[i])) < 1e-8


def test_choices_by_hand():
    l = torch.tensor([[3.0, 0, 2, 2, 1, 1, 2.5, -9]])
    assert choose(l, 4, 2, 3).tolist() == [[0, 6, 1]]            # groups of two: 0 (3.0) and 3 (2.5)
    # sums of two sigmoids: 1.453, 1.762, 1.462, 0.924
    assert choose(l, 4, 2, 3, scoring="sigmoid").tolist() == [[2, 3, 4]]
    tie = torch.zeros(1, 8)
    assert choose(tie, 4, 2, 4).tolist() == [[0, 1, 2, 3]] and choose(tie, 2, 1, 2, scoring="sigmoid").tolist() == [[0, 1]]
    bias = torch.tensor([0.0, 0, 0, 0, 0, 0, 0.1, 0.1])
    assert choose(tie, 4, 1, 2, bias, "sigmoid").tolist() == [[6, 7]]
