"""e4m3 weights that the tensor cores cannot read in place are refused, not copied on every call."""
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


def fp8(*shape, offset=0, block_rows=128):
    """Values `offset` bytes behind a multiple of 16, as a file mapped at an odd place has them."""
    n = torch.Size(shape).numel()
    raw = torch.zeros(n + 64, dtype=torch.uint8)
    start = -raw.data_ptr() % 16 + offset
    q = raw[start:start + n].view(F8).view(shape)
    assert q.data_ptr() % 16 == offset % 16
    return nob.Fp8(q, torch.ones(*shape[:-2], -(-shape[-2] // block_rows), -(-shape[-1] // 128)))


def calls(p, offset):
    x, idx, w = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    return {
        "w": lambda: p.matmul_fp8(fp8(3, 256, block_rows=1), fp8(5, 256, offset=offset)),
        "gate_up": lambda: p.experts_fp8(x, fp8(8, 2, 64, 256, offset=offset), fp8(8, 256, 64), idx, w),
        "down": lambda: p.experts_fp8(x, fp8(8, 2, 64, 256), fp8(8, 256, 64, offset=offset), idx, w),
    }


@pytest.mark.parametrize("name", ["w", "gate_up", "down"])
def test_weights_that_are_not_aligned_are_refused(plane, name):
    for offset in (1, 4, 8):
        with pytest.raises(ValueError, match=name + ".q must be 16-byte aligned"):
            calls(plane, offset)[name]()
    with pytest.raises(MoEError, match="null context"):
        calls(plane, 16)[name]()


def test_rows_that_are_not_aligned_are_taken(plane):
    """Activations, a call's own small operand, are copied to an aligned place."""
    with pytest.raises(MoEError, match="null context"):
        plane.matmul_fp8(fp8(3, 256, offset=1, block_rows=1), fp8(5, 256))
