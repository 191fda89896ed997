"""What the e4m3 and balance-loss calls refuse, without a GPU: the Python checks with tensors of the host,
the C entry points with a null context."""
import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200 import _lib
from npu_offload_b200._lib import MoEError

F8 = torch.float8_e4m3fn


@pytest.fixture
def plane(monkeypatch):
    """A plane of the host's memory whose C calls get a null context."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    return p


def fp8(*shape, block_rows=128):
    return nob.Fp8(torch.zeros(shape).to(F8), torch.ones(*shape[:-2], -(-shape[-2] // block_rows), -(-shape[-1] // 128)))


def reaches_the_library(call):
    with pytest.raises(MoEError, match="null context"):
        call()


@pytest.mark.parametrize("x,kw,needle", [
    (torch.zeros(4, 32, dtype=torch.float16), {}, "float16"),
    (torch.zeros(32), {}, "rows, cols"),
    (torch.zeros(4, 32), dict(block_rows=64), "block_rows"),
    ([1.0], {}, "tensor on"),
])
def test_quantize_refuses(plane, x, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.quantize_fp8(x, **kw)


def test_quantize_takes_what_is_documented(plane):
    for x in (torch.zeros(4, 32), torch.zeros(2, 3, 32, dtype=torch.bfloat16), torch.zeros(32, 4).T, torch.zeros(0, 32)):
        reaches_the_library(lambda: plane.quantize_fp8(x))


@pytest.mark.parametrize("x,w,kw,needle", [
    (fp8(3, 32, block_rows=1), fp8(5, 48), {}, "columns"),
    (fp8(3, 32, block_rows=1), torch.zeros(5, 32), {}, "Fp8"),
    (fp8(3, 32, block_rows=1), fp8(2, 5, 32), {}, "dimensions"),
    (fp8(3, 32, block_rows=128), fp8(5, 32), {}, "x.scale"),
    (fp8(3, 32, block_rows=1), fp8(300, 32, block_rows=64), {}, "w.scale"),
    (fp8(3, 32, block_rows=1), nob.Fp8(torch.zeros(32, 16).to(F8).T, torch.ones(1, 1)), {}, "contiguous"),
    (fp8(3, 32, block_rows=1), fp8(5, 32), dict(out_dtype=torch.float16), "out_dtype"),
    (fp8(3, 32, block_rows=1), fp8(5, 32), dict(out=torch.zeros(3, 4)), "out must be"),
    (fp8(3, 32, block_rows=1), fp8(5, 32), dict(out=torch.zeros(5, 3).T), "out must be"),
])
def test_matmul_refuses(plane, x, w, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.matmul_fp8(x, w, **kw)


def expert_args(**kw):
    a = dict(x=torch.zeros(3, 256, dtype=torch.bfloat16), gate_up=fp8(8, 2, 64, 256), down=fp8(8, 256, 64),
             idx=torch.zeros(3, 2, dtype=torch.int32), w=torch.zeros(3, 2))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,needle", [
    (dict(x=torch.zeros(3, 256)), "float32"),
    (dict(x=torch.zeros(3, 128, dtype=torch.bfloat16)), "columns"),
    (dict(gate_up=fp8(8, 128, 256)), "dimensions"),
    (dict(gate_up=fp8(7, 2, 64, 256)), "gate_up is"),
    (dict(down=fp8(8, 64, 256)), "down is"),
    (dict(idx=torch.zeros(3, 2, dtype=torch.int64)), "int64"),
    (dict(idx=torch.zeros(3, 1, dtype=torch.int32)), "must be"),
    (dict(w=torch.zeros(2, 2)), "must be"),
    (dict(accumulate=True), "accumulate"),
    (dict(out=torch.zeros(3, 128)), "out must be"),
])
def test_experts_refuse(plane, kw, needle):
    with pytest.raises(ValueError, match=needle):
        plane.experts_fp8(**expert_args(**kw))


@pytest.mark.parametrize("kw,needle", [
    (dict(logits=torch.zeros(4, 7)), "columns"),
    (dict(logits=torch.zeros(4, 8, dtype=torch.bfloat16)), "bfloat16"),
    (dict(logits=torch.zeros(4, 8, requires_grad=True)), "autograd"),
    (dict(idx=torch.zeros(4, 3, dtype=torch.int32)), "idx is"),
    (dict(offsets=torch.zeros(1, dtype=torch.int32)), "two entries"),
    (dict(offsets=torch.zeros(3, dtype=torch.int64)), "int64"),
    (dict(mask=torch.ones(5, dtype=torch.bool)), "mask has"),
    (dict(mask=torch.ones(4)), "mask is"),
])
def test_balance_refuses(plane, kw, needle):
    a = dict(logits=torch.zeros(4, 8), idx=torch.zeros(4, 2, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(ValueError, match=needle):
        plane.balance_loss(**a)


def test_balance_backward_refuses(plane):
    lg = torch.zeros(4, 8)
    st = nob.BalanceStats(torch.zeros(1, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), None, None)
    for bad in (st._replace(counts=torch.zeros(2, 8, dtype=torch.int32)), st._replace(tokens=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="other sequences"):
            plane.balance_loss_backward(lg, bad)
    with pytest.raises(ValueError, match="grad has"):
        plane.balance_loss_backward(lg, st, grad=torch.ones(1))
    reaches_the_library(lambda: plane.balance_loss_backward(lg, st, grad=torch.ones(())))
    with torch.no_grad():
        reaches_the_library(lambda: plane.balance_loss(lg.requires_grad_(), torch.zeros(4, 2, dtype=torch.int32)))


def test_c_entry_points_report_a_null_context():
    L = nob.lib()
    assert L.moe_quantize_fp8(None, None, 0, 1, 1, 16, 1, None, None, 0, None) == _lib.MOE_EINVAL
    assert L.moe_matmul_fp8(None, 1, 1, 16, None, None, None, None, None, 0, 0, None) == _lib.MOE_EINVAL
    assert L.moe_experts_fp8_workspace(None, 1) == -1
    assert L.moe_experts_fp8(None, 1, *[None] * 8, 0, None, 0, 0, None) == _lib.MOE_EINVAL
    assert L.moe_balance_loss_workspace(None, 1, 1) == -1
    assert L.moe_balance_loss(None, 1, None, None, None, 1, None, None, None, None, None, 0, 0, None) == _lib.MOE_EINVAL
    assert L.moe_balance_loss_backward(None, 1, None, None, 1, None, None, None, None, None, 0, None) == _lib.MOE_EINVAL


def test_definitions_agree_on_the_host():
    """The 64-bit quantiser of the tests against torch's own e4m3 conversion, and the balance gradient
    against differences."""
    from tests.fp8_util import balance64, expand, quantize64
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 272, generator=g) * torch.exp(3 * torch.randn(5, 1, generator=g))
    x[2] = 0
    x[3, 7] = float("inf")
    q, s = quantize64(x, 1)
    ref = (x / expand(s, x.shape, 1).float()).to(F8).double()
    assert torch.equal(torch.nan_to_num(q, nan=1e9), torch.nan_to_num(ref, nan=1e9))
    assert (s[2] == 1).all() and q[3, 7].isnan()
    off = torch.tensor([0, 2, 2, 6])
    for scoring in ("softmax", "sigmoid"):
        l = torch.randn(7, 5, generator=g, dtype=torch.float64)
        idx = l.topk(2, -1)[1].int()
        mask = torch.tensor([1, 1, 1, 0, 1, 1, 1], dtype=torch.bool)
        loss, counts, d = balance64(l, idx, off, mask, scoring)
        assert counts.sum() == 2 * 5 and (d[3] == 0).all() and (d[6] == 0).all()
        for t in range(7):
            for e in range(5):
                h = torch.zeros_like(l)
                h[t, e] = 1e-5
                num = (balance64(l + h, idx, off, mask, scoring)[0] - balance64(l - h, idx, off, mask, scoring)[0]) / 2e-5
                assert abs(float(num - d[t, e])) < 1e-9
