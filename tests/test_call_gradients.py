"""Calls without a backward pass refuse operands that require a gradient instead of dropping it in silence."""
import pytest
import torch

import npu_offload_b200 as nob
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


def experts(p, **kw):
    a = dict(x=torch.zeros(3, 256, dtype=torch.bfloat16), gate_up=fp8(8, 2, 64, 256), down=fp8(8, 256, 64),
             idx=torch.zeros(3, 2, dtype=torch.int32), w=torch.zeros(3, 2))
    a.update(kw)
    return p.experts_fp8(**a)


def leaf(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, requires_grad=True)


def scaled(m):
    return m._replace(scale=m.scale.requires_grad_())


ROWS = fp8(3, 32, block_rows=1)
STATS = nob.BalanceStats(torch.zeros(1, 8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), None, None)
CALLS = {
    "quantize x": lambda p: p.quantize_fp8(leaf(4, 32)),
    "quantize x as a view": lambda p: p.quantize_fp8(leaf(32, 4).T),
    "matmul x": lambda p: p.matmul_fp8(leaf(3, 32), fp8(5, 32)),
    "matmul x.scale": lambda p: p.matmul_fp8(scaled(fp8(3, 32, block_rows=1)), fp8(5, 32)),
    "matmul w.scale": lambda p: p.matmul_fp8(ROWS, scaled(fp8(5, 32))),
    "matmul out": lambda p: p.matmul_fp8(ROWS, fp8(5, 32), out=leaf(3, 5)),
    "experts x": lambda p: experts(p, x=leaf(3, 256, dtype=torch.bfloat16)),
    "experts w": lambda p: experts(p, w=leaf(3, 2)),
    "experts gate_up": lambda p: experts(p, gate_up=scaled(fp8(8, 2, 64, 256))),
    "experts down": lambda p: experts(p, down=scaled(fp8(8, 256, 64))),
    "experts out": lambda p: experts(p, out=leaf(3, 256)),
    "route logits": lambda p: p.route_topk(leaf(3, 8)),
    "balance out": lambda p: p.balance_loss_backward(torch.zeros(4, 8), STATS, out=leaf(4, 8)),
    "balance grad": lambda p: p.balance_loss_backward(torch.zeros(4, 8), STATS, grad=leaf(())),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_an_operand_that_requires_a_gradient_is_refused(plane, name):
    with pytest.raises(ValueError, match="autograd"):
        CALLS[name](plane)


def test_a_correction_bias_only_selects(plane):
    """The weights are those of the scores without it: a bias that is a parameter loses nothing."""
    with pytest.raises(MoEError, match="null context"):
        plane.route_topk(torch.zeros(3, 8), leaf(8))


@pytest.mark.parametrize("name", list(CALLS))
def test_it_is_taken_where_nothing_records(plane, name):
    with torch.no_grad(), pytest.raises(MoEError, match="null context"):
        CALLS[name](plane)
