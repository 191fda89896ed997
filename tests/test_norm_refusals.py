"""What the norm's calls refuse and take, without a GPU; the 64-bit definition against differences."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200 import _lib
from npu_offload_b200._lib import MoEError
from tests.norm_util import norm64, norm_backward64, scales64


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


X, W = torch.zeros(3, 32), torch.ones(32)


@pytest.mark.parametrize("kw,needle", [
    (dict(x=torch.zeros(3, 32, dtype=torch.float16)), "float16"),
    (dict(x=torch.zeros(())), "column"),
    (dict(x=torch.zeros(3, 0), weight=torch.ones(0)), "column"),
    (dict(x=[1.0]), "tensor on"),
    (dict(weight=torch.ones(31)), "weight has"),
    (dict(weight=torch.ones(1, 32)), "dimensions"),
    (dict(weight=torch.ones(32, dtype=torch.float64)), "float64"),
    (dict(weight=None), "tensor on"),
    (dict(residual=torch.zeros(2, 32)), "residual is"),
    (dict(residual=torch.zeros(3, 32, dtype=torch.float16)), "float16"),
    (dict(out_dtype=torch.float16), "out_dtype"),
    (dict(out_dtype=None), "neither"),
    (dict(x=torch.zeros(3, 24), weight=torch.ones(24), fp8=True), "multiple of 16"),
    (dict(x=torch.zeros(3, 32, requires_grad=True)), "autograd"),
    (dict(weight=torch.ones(32, requires_grad=True)), "autograd"),
    (dict(residual=torch.zeros(3, 32, requires_grad=True)), "autograd"),
])
def test_add_norm_refuses(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.add_norm(**{**dict(x=X, weight=W), **kw})


@pytest.mark.parametrize("kw", [
    dict(), dict(residual=torch.zeros(3, 32, dtype=torch.bfloat16)), dict(fp8=True), dict(fp8=True, out_dtype=None),
    dict(out_dtype=torch.float32), dict(x=torch.zeros(2, 3, 32)), dict(x=torch.zeros(32)), dict(x=torch.zeros(0, 32)),
    dict(x=torch.zeros(32, 3).T), dict(weight=W.to(torch.bfloat16)),
])
def test_add_norm_takes_what_is_documented(plane, kw):
    reaches_the_library(lambda: plane.add_norm(**{**dict(x=X, weight=W), **kw}))


@pytest.mark.parametrize("kw,needle", [
    (dict(dy=torch.zeros(2, 32)), "dy is"),
    (dict(dy=torch.zeros(3, 32, dtype=torch.float64)), "float64"),
    (dict(sum=torch.zeros(3, 32, dtype=torch.float16)), "float16"),
    (dict(weight=torch.ones(31)), "weight has"),
    (dict(rstd=torch.ones(2)), "rstd is"),
    (dict(rstd=torch.ones(3, 1)), "dimensions"),
    (dict(rstd=torch.ones(3, dtype=torch.float64)), "float64"),
    (dict(dsum=torch.zeros(3, 31)), "dsum is"),
    (dict(dsum=torch.zeros(3, 32, dtype=torch.bfloat16)), "bfloat16"),
    (dict(dy=torch.zeros(3, 32, requires_grad=True)), "autograd"),
    (dict(sum=torch.zeros(3, 32, requires_grad=True)), "autograd"),
])
def test_backward_refuses(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.add_norm_backward(**{**dict(dy=X, sum=X, weight=W, rstd=torch.ones(3)), **kw})


def test_backward_takes_what_is_documented(plane):
    a = dict(dy=X.to(torch.bfloat16), sum=X, weight=W, rstd=torch.ones(3), dsum=X)
    reaches_the_library(lambda: plane.add_norm_backward(**a))
    reaches_the_library(lambda: plane.add_norm_backward(**a, weight_grad=False))
    with torch.no_grad():
        reaches_the_library(lambda: plane.add_norm(X, W.clone().requires_grad_()))


def test_a_stream_of_another_device_is_refused(plane, monkeypatch):
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    plane.device = torch.device("cuda", 0)
    other = SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=5)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        plane.add_norm(X, W, stream=other)
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        plane.add_norm_backward(X, X, W, torch.ones(3), stream=other)


def test_c_entry_points_report_a_null_context():
    L = nob.lib()
    assert L.moe_add_norm(None, 1, 16, None, 0, None, 0, None, 0, 1e-6, None, None, 0, None, None, None, 0, None) == _lib.MOE_EINVAL
    assert L.moe_add_norm_backward_workspace(None, 1, 16) == -1
    assert L.moe_add_norm_backward(None, 1, 16, None, 0, None, 0, None, None, 0, None, None, None, None, 0, 0, None) == _lib.MOE_EINVAL


def test_the_gradient_agrees_with_differences():
    g = torch.Generator().manual_seed(3)
    h, w, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 7), (7,), (3, 7)))
    eps, step = 1e-3, 1e-6
    _, rstd = norm64(h, w, eps)
    dx, dw, _, _ = norm_backward64(dy, h, w, rstd)
    f = lambda h, w: (norm64(h, w, eps)[0] * dy).sum()  # noqa: E731
    for i in range(h.numel()):
        d = torch.zeros_like(h)
        d.view(-1)[i] = step
        assert abs(float((f(h + d, w) - f(h - d, w)) / (2 * step) - dx.view(-1)[i])) < 1e-8
    for i in range(7):
        d = torch.zeros_like(w)
        d[i] = step
        assert abs(float((f(h, w + d) - f(h, w - d)) / (2 * step) - dw[i])) < 1e-8


def test_scales_by_their_definition():
    y = torch.zeros(1, 128 * 5, dtype=torch.float64)
    for i, v in enumerate((448.0, 448.0000001, 2.0 ** -140, 3.5, 0.0)):
        y[0, 128 * i + i] = -v
    assert scales64(y)[0].tolist() == [1.0, 2.0, 2.0 ** -126, 2.0 ** -7, 1.0]
