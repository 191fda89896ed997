"""The norm in rows that are no multiples of eight values, whose first and last words hold their neighbours' values: squares out of
range, NaN and infinities next door, and the gradients of the same.  Tolerances as the norm's other tests derive them."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.norm_util import norm64, norm_backward64, rounded_sum

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
WORK = 2.0 ** -19
COLS = [1, 3, 7, 9, 100, 641, 1283, 2047, 2049, 4095, 4099, 8193, 12289, 16381]


@pytest.fixture(scope="module")
def plane():
    with nob.MoEDataPlane(256, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        yield p


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(t):
    return torch.finfo(t).eps / 2


@pytest.mark.parametrize("C", COLS + [640, 4096, 12288])
@pytest.mark.parametrize("size,eps", [(1e25, 1e-6), (1e-25, 1e-30), (3e38, 1e-6), (1e-18, 1e-37)])
@pytest.mark.parametrize("x_dtype,r_dtype", [(BF, None), (F32, None), (BF, BF), (F32, F32)])
def test_squares_that_leave_the_range(plane, C, size, eps, x_dtype, r_dtype):
    """Such rows and ordinary ones in turn."""
    g = gen(C)
    x = torch.rand(9, C, generator=g, device="cuda") * 2 - 1
    x[::2] *= size / (2 if r_dtype else 1)
    x = x.to(x_dtype)
    r = None if r_dtype is None else (x.float() * torch.rand(9, C, generator=g, device="cuda")).to(r_dtype)
    w = 1 + 0.3 * torch.randn(C, generator=g, device="cuda").clamp(-2, 2)
    n = plane.add_norm(x, w, r, eps=eps, out_dtype=F32)
    h = rounded_sum(x, r)
    assert torch.equal(n.sum, h)
    y, rstd = norm64(h, w, float(torch.tensor(eps, dtype=F32)))
    assert ((n.y.double() - y).abs() <= (half_step(F32) + WORK) * y.abs() + 1e-40).all()
    assert ((n.rstd.double() - rstd).abs() <= WORK * rstd + 2.0 ** -149).all()


@pytest.mark.parametrize("C", COLS)
@pytest.mark.parametrize("T", [9, 700])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_special_values_stay_in_their_row(plane, C, T, dtype):
    g = gen(C + T)
    x, r = torch.randn(T, C, generator=g, device="cuda").to(dtype), torch.randn(T, C, generator=g, device="cuda").to(dtype)
    w = 1 + 0.3 * torch.randn(C, generator=g, device="cuda")
    dy, rstd = torch.randn(T, C, generator=g, device="cuda").to(dtype), 0.5 + torch.rand(T, generator=g, device="cuda")
    bad = torch.zeros(T, dtype=torch.bool, device="cuda")
    bad[1::3] = True
    clean = plane.add_norm(x, w, r, out_dtype=F32)
    want, want_w = plane.add_norm_backward(dy, x, w, rstd, dsum=r)
    for value in (float("nan"), float("inf"), -float("inf")):
        xs, dys, sums = x.clone(), dy.clone(), x.clone()
        xs[bad], dys[bad] = value, value
        n = plane.add_norm(xs, w, r, out_dtype=F32)
        for got, was in ((n.y, clean.y), (n.sum, clean.sum), (n.rstd, clean.rstd)):
            assert torch.equal(got[~bad], was[~bad])
        assert n.y[bad].isnan().all()  # rstd is 0 or NaN, times an infinity or NaN
        sums[bad] = value
        dx, dw = plane.add_norm_backward(dys, sums, w, rstd, dsum=r)
        assert torch.equal(dx[~bad], want[~bad]) and not dx[bad].isfinite().any() and not dw.isfinite().any()
    # rows of nothing but zeros between rows of large values: their gradient is the weight's alone
    dy0 = dy.clone()
    dy0[bad] = 0
    dx, dw = plane.add_norm_backward(dy0, x, w, rstd)
    exact, exact_w, size, size_w = norm_backward64(dy0, x, w, rstd)
    assert (dx[bad] == 0).all() and ((dx.double() - exact).abs() <= half_step(dtype) * exact.abs() + 2 * WORK * size + 1e-40).all()
    assert ((dw.double() - exact_w).abs() <= WORK * size_w + 1e-40).all()


@pytest.mark.parametrize("C", [4097, 4098, 4100, 4099, 5121, 8191])
def test_no_more_ctas_than_run_at_once(plane, C):
    """Rows of that length have one CTA an SM, whose shares of the weight's gradient the workspace holds: a CTA more would run behind all others."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for T in (1, 100, sms, sms + 1, 1000, 4000, 8192, 16384, 65536):
        n = nob.lib().moe_add_norm_backward_workspace(plane.handle, T, C)
        assert n % (4 * C) == 0 and 1 <= n // (4 * C) <= min(sms, T)
