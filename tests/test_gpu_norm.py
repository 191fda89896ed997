"""Residual addition with root-mean-square norm, and its gradients, against 64 bits.

Tolerances (steps of 2^-24, relative): the sum of squares is of positive terms, 16 of them one after the other on a thread
and 10 levels of additions behind that, so off by 26 at most, half of which reach rstd; its root is off by 2 steps of
2^-23 and the mean's division and addition by one step each, the two products by one each: 13 + 4 + 1 + 2 = 20 < 2^-19.
A result is then rounded once, by half a step of its type."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.norm_util import norm64, norm_backward64, rounded_sum, scales64

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
WORK = 2.0 ** -19


@pytest.fixture(scope="module")
def plane():
    with nob.MoEDataPlane(256, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        yield p


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(g, *shape, dtype=F32):
    return (torch.randn(*shape, generator=g, device="cuda") * torch.exp(torch.randn(*shape[:-1], 1, generator=g, device="cuda"))).to(dtype)


def half_step(t):
    return torch.finfo(t).eps / 2


def check(n, x, w, residual, eps, out_dtype, fp8):
    h = rounded_sum(x, residual)
    if residual is None:
        assert n.sum is x or torch.equal(n.sum, x)
    else:
        assert n.sum.dtype == residual.dtype and torch.equal(n.sum, h)
    y, rstd = norm64(h, w, eps)
    assert n.rstd.shape == x.shape[:-1]
    assert ((n.rstd.double() - rstd).abs() <= WORK * rstd).all()
    assert (n.y is None) == (out_dtype is None) and (n.fp8 is None) == (not fp8)
    if out_dtype is not None:
        assert n.y.dtype == out_dtype and n.y.shape == x.shape
        assert ((n.y.double() - y).abs() <= (half_step(out_dtype) + WORK) * y.abs() + 1e-40).all()
    if fp8:
        s = scales64(y)
        assert torch.equal(n.fp8.scale.double(), s)
        s = s.repeat_interleave(128, -1)[..., : y.shape[-1]]
        # rounded by half a step: 2^-4 of the value, 2^-10 scales at the bottom of the range
        assert ((n.fp8.q.double() * s - y).abs() <= (2.0 ** -4 + 2 * WORK) * y.abs() + 2.0 ** -10 * s).all()


SHAPES = [(1, 1), (1, 16), (6, 144), (150, 1040), (4, 2064), (149, 4112), (3, 8176), (3, 8), (5, 7), (2, 127), (7, 128), (4, 129), (9, 1000), (33, 1280), (17, 1283), (300, 2048), (5, 2056), (1, 4096),
          (700, 4096), (3, 4100), (2, 8192), (2, 8200), (3, 8193), (2, 16384), (1, 16383), (9, 16381), (400, 130), (1000, 2047), (301, 4095), (600, 4), (5000, 3), (333, 1)]


@pytest.mark.parametrize("T,C", SHAPES)
@pytest.mark.parametrize("x_dtype,r_dtype", [(BF, BF), (F32, BF), (BF, F32), (F32, F32), (BF, None), (F32, None)])
def test_forward(plane, T, C, x_dtype, r_dtype):
    g = gen(T * 31 + C)
    x, w = rows(g, T, C, dtype=x_dtype), 1 + 0.3 * torch.randn(C, generator=g, device="cuda")
    r = None if r_dtype is None else rows(g, T, C, dtype=r_dtype)
    fp8 = C % 16 == 0
    for out, wt in ((BF, w.to(BF)), (F32, w)):
        check(plane.add_norm(x, wt, r, eps=1e-5, out_dtype=out, fp8=fp8), x, wt, r, 1e-5, out, fp8)
    if fp8:
        check(plane.add_norm(x, w, r, eps=1e-5, out_dtype=None, fp8=True), x, w, r, 1e-5, None, True)


@pytest.mark.parametrize("T,C", SHAPES)
@pytest.mark.parametrize("dy_dtype,s_dtype,with_dsum", [(BF, BF, True), (BF, BF, False), (F32, F32, False), (F32, BF, True), (BF, F32, True), (F32, F32, True),
                                                        (F32, BF, False), (BF, F32, False)])
def test_backward(plane, T, C, dy_dtype, s_dtype, with_dsum):
    """dx: every term of the formula is off by the work's few steps of its own size (C of them in the mean: 26 steps), the
    result by half a step.  dweight: rows after one another on a CTA (12 at most here), then at most 14 shares and 5 levels."""
    g = gen(T * 17 + C)
    h, dy = rows(g, T, C, dtype=s_dtype), rows(g, T, C, dtype=dy_dtype)
    w = (1 + 0.3 * torch.randn(C, generator=g, device="cuda")).to(BF if T % 2 else F32)
    ds = rows(g, T, C, dtype=s_dtype) if with_dsum else None
    rstd = norm64(h, w, 1e-5)[1].float()
    want, want_w, size, size_w = norm_backward64(dy, h, w, rstd, ds)
    dx, dw = plane.add_norm_backward(dy, h, w, rstd, dsum=ds)
    assert dx.dtype == s_dtype and dw.dtype == F32 and dw.shape == (C,)
    assert ((dx.double() - want).abs() <= half_step(s_dtype) * want.abs() + 2 * WORK * size + 1e-40).all()
    assert ((dw.double() - want_w).abs() <= WORK * size_w + 1e-40).all()
    again, none = plane.add_norm_backward(dy, h, w, rstd, dsum=ds, weight_grad=False)
    assert none is None and torch.equal(again, dx)
    assert torch.equal(plane.add_norm_backward(dy, h, w, rstd, dsum=ds)[1], dw)  # no sum depends on timing


def test_many_rows(plane):
    """More rows than a wave; dweight: 66 rows after one another on a CTA, 5 shares, 5 levels: 76 + 3 steps < 2^-17."""
    g = gen(5)
    T, C = 19531, 512
    x, r, w = rows(g, T, C, dtype=BF), rows(g, T, C, dtype=BF), torch.ones(C, device="cuda", dtype=BF)
    n = plane.add_norm(x, w, r, eps=1e-6, fp8=True)
    check(n, x, w, r, 1e-6, BF, True)
    dy = rows(g, T, C, dtype=BF)
    dx, dw = plane.add_norm_backward(dy, n.sum, w, n.rstd)
    want, want_w, size, size_w = norm_backward64(dy, n.sum, w, n.rstd)
    assert ((dx.double() - want).abs() <= half_step(BF) * want.abs() + 2 * WORK * size).all()
    assert ((dw.double() - want_w).abs() <= 2.0 ** -17 * size_w).all()


@pytest.mark.parametrize("kind", [BF, F32])
def test_scales_at_their_borders(plane, kind):
    """The largest value of each group within a few steps of 448 2^k, either side: the scale is the definition's."""
    g = gen(9)
    for trial in range(12):
        h = rows(g, 1, 4096, dtype=kind)
        rstd = norm64(h, torch.ones(4096, device="cuda"), 1e-6)[1]
        w = torch.full((4096,), 1e-3, device="cuda", dtype=torch.float64)
        at = torch.arange(32, device="cuda") * 128 + h.double().abs().view(32, 128).argmax(-1)
        delta = (torch.arange(32, device="cuda", dtype=torch.float64) - 16) * (2.0 ** -24 if trial % 2 else 2.0 ** -26)
        w[at] = 448 * 2.0 ** (trial - 6) * (1 + delta) / (h[0, at].double().abs() * rstd)
        w = w.float()
        check(plane.add_norm(h, w, eps=1e-6, fp8=True), h, w, None, 1e-6, BF, True)


@pytest.mark.parametrize("size,eps", [(1e25, 1e-6), (1e-25, 1e-30), (3e38, 1e-6), (1e-30, 1e-6), (1e-18, 1e-37)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_squares_that_leave_the_range(plane, size, eps, dtype):
    g = gen(2)
    x = (torch.rand(5, 640, generator=g, device="cuda") * 2 - 1).mul(size).to(dtype)
    w = torch.ones(640, device="cuda")
    n = plane.add_norm(x, w, eps=eps, out_dtype=F32)
    y, rstd = norm64(x, w, float(torch.tensor(eps, dtype=F32)))
    assert ((n.y.double() - y).abs() <= (half_step(F32) + WORK) * y.abs() + 1e-40).all()
    assert ((n.rstd.double() - rstd).abs() <= WORK * rstd + 2.0 ** -149).all()


def test_rows_of_zeros_and_special_values(plane):
    g = gen(4)
    x = rows(g, 6, 256)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 200] = float("nan")
    x[4, 3] = -float("inf")
    w = torch.ones(256, device="cuda")
    n = plane.add_norm(x, w, eps=1e-6, out_dtype=F32, fp8=True)
    keep = [0, 1, 5]
    check(nob.moe.Normed(n.y[keep], nob.Fp8(n.fp8.q[keep], n.fp8.scale[keep]), x[keep], n.rstd[keep]), x[keep], w, None, 1e-6, F32, True)
    assert (n.y[1] == 0).all() and (n.fp8.scale[1] == 1).all()
    want, _ = norm64(x, w, 1e-6)
    for t in (2, 3, 4):
        assert torch.equal(n.y[t].isnan(), want[t].isnan()) and torch.equal(n.fp8.q[t].float().isnan(), want[t].isnan())
        fine = ~want[t].isnan()
        assert (n.y[t][fine] == 0).all()


def test_strides_and_alignment(plane):
    g = gen(6)
    big = rows(g, 9, 2 * 256)
    x, r = big[:, :256], rows(g, 256, 9, dtype=BF).T
    w = torch.ones(257, device="cuda")[1:]  # not at a 16-byte boundary
    check(plane.add_norm(x, w, r, eps=1e-5, fp8=True), x, w, r, 1e-5, BF, True)
    odd = rows(g, 9 * 256 + 1, 1).reshape(-1)[1:].view(9, 256)
    n = plane.add_norm(odd, w, r, eps=1e-5, fp8=True)
    check(n, odd, w, r, 1e-5, BF, True)
    dy = rows(g, 256, 9, dtype=BF).T
    a = plane.add_norm_backward(dy, n.sum, w, n.rstd, dsum=r)
    b = plane.add_norm_backward(dy.contiguous(), n.sum, w.clone(), n.rstd, dsum=r.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows_and_leading_dimensions(plane):
    w = torch.ones(32, device="cuda")
    n = plane.add_norm(torch.zeros(0, 32, device="cuda"), w, torch.zeros(0, 32, device="cuda", dtype=BF), fp8=True)
    assert n.y.shape == n.sum.shape == n.fp8.q.shape == (0, 32) and n.rstd.shape == (0,) and n.fp8.scale.shape == (0, 1)
    dx, dw = plane.add_norm_backward(torch.zeros(0, 32, device="cuda"), torch.zeros(0, 32, device="cuda"), w, n.rstd)
    assert dx.shape == (0, 32) and (dw == 0).all()
    g = gen(7)
    x = rows(g, 2, 3, 32)
    a, b = plane.add_norm(x, w, fp8=True), plane.add_norm(x.view(6, 32), w, fp8=True)
    assert a.y.shape == (2, 3, 32) and a.rstd.shape == (2, 3) and a.fp8.scale.shape == (2, 3, 1) and torch.equal(a.y.view(6, 32), b.y)
    lone = plane.add_norm(x[0, 0], w)
    assert lone.y.shape == (32,) and lone.rstd.shape == () and torch.equal(lone.y, a.y[0, 0])


def test_the_norm_feeds_the_product(plane):
    """Fp8 rows straight into matmul_fp8: the same as through quantize_fp8 of the fp32 rows, but for values that the
    product of three factors puts on another side of a rounding border."""
    g = gen(8)
    x, w = rows(g, 37, 512, dtype=BF), (1 + 0.2 * torch.randn(512, generator=g, device="cuda")).to(BF)
    m = plane.quantize_fp8(torch.randn(200, 512, generator=g, device="cuda") * 0.05, block_rows=128)
    n = plane.add_norm(x, w, out_dtype=F32, fp8=True)
    q = plane.quantize_fp8(n.y)
    assert torch.equal(q.scale, n.fp8.scale) and torch.equal(q.q.view(torch.uint8), n.fp8.q.view(torch.uint8))
    assert torch.equal(plane.matmul_fp8(n.fp8, m), plane.matmul_fp8(q, m))


def test_another_stream_and_captured_graphs(plane):
    g = gen(11)
    data = [(rows(g, 50, 1280, dtype=BF), rows(g, 50, 1280, dtype=BF), torch.ones(1280, device="cuda", dtype=BF), rows(g, 50, 1280, dtype=BF)) for _ in range(2)]

    def step(x, r, w, dy, stream=None):
        n = plane.add_norm(x, w, r, fp8=True, stream=stream)
        return (n.y, n.fp8.q.view(torch.uint8), n.fp8.scale, n.sum, n.rstd, *plane.add_norm_backward(dy, n.sum, w, n.rstd, dsum=r, stream=stream))

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = step(*data[0], stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
    streams, graphs, outs = [torch.cuda.Stream() for _ in data], [], []
    for s, d in zip(streams, data):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(step(*d))
        graphs.append(graph)
    for _ in range(10):
        for s, graph, o in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                o[0].zero_(), o[-1].zero_()
                graph.replay()
    torch.cuda.synchronize()
    for o, v in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, v))


def test_the_c_calls_refuse_what_would_overlap(plane):
    """Arguments that the library's own checks turn away; nothing is launched."""
    from npu_offload_b200 import _lib
    L, x = nob.lib(), torch.zeros(4, 32, device="cuda")
    w, rstd, p = torch.ones(32, device="cuda"), torch.ones(4, device="cuda"), lambda t: t.data_ptr()
    before = plane.launch_count

    def call(T=4, C=32, xp=p(x), res=None, eps=1e-6, total=None, y=None, q=None, s=None, flags=0):
        return L.moe_add_norm(plane.handle, T, C, xp, 1, res, 1, p(w), 1, eps, total, y, 1, q, s, p(rstd), flags, None)

    z = torch.zeros(4, 32, device="cuda")
    for kw, needle in ((dict(T=-1), "T="), (dict(T=1 << 25), "T="), (dict(C=0), "C="), (dict(C=16385), "C="), (dict(y=p(x)), "overlaps"),
                       (dict(res=p(z), total=p(z)), "overlaps"), (dict(res=p(z)), "together"), (dict(q=p(z)), "together"),
                       (dict(C=24, q=p(z), s=p(z)), "multiple of 16"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
                       (dict(eps=float("inf")), "eps"), (dict(y=p(z), q=p(z) + 1024, s=p(rstd) + 2), "4-byte"), (dict(flags=1), "flag"), (dict(xp=p(x) + 4), "aligned"), (dict(xp=None), "null")):
        assert call(**kw) == _lib.MOE_EINVAL and needle in _lib.last_error(), kw
    dw, ws = torch.zeros(32, device="cuda"), torch.zeros(1 << 20, device="cuda")

    def back(dx=p(z), dweight=p(dw), work=p(ws), n=1 << 22):
        return L.moe_add_norm_backward(plane.handle, 4, 32, p(x), 1, p(x), 1, None, p(w), 1, p(rstd), dx, dweight, work, n, 0, None)

    for kw, needle in ((dict(dx=p(x)), "overlaps"), (dict(dx=None), "null"), (dict(work=None), "workspace"), (dict(n=8), "workspace"),
                       (dict(work=p(ws) + 16), "workspace")):
        assert back(**kw) == _lib.MOE_EINVAL and needle in _lib.last_error(), kw
    assert plane.launch_count == before


def test_the_weights_gradient_overlaps_nothing(plane):
    """dweight on an operand: written while other rows may still be read.  Nothing is launched."""
    from npu_offload_b200 import _lib
    L, f = nob.lib(), lambda *shape: torch.zeros(*shape, device="cuda")
    dy, total, dsum, w, rstd, dx, ws = f(4, 32), f(4, 32), f(4, 32), f(32), f(64), f(4, 32), f(1 << 20)
    p, before = lambda t: t.data_ptr(), plane.launch_count
    for t in (dy, total, dsum, w, rstd, dx):
        for at in (p(t), p(t) + 4, p(t) - 124):
            assert L.moe_add_norm_backward(plane.handle, 4, 32, p(dy), 1, p(total), 1, p(dsum), p(w), 1, p(rstd), p(dx), at, p(ws), 1 << 22,
                                           0, None) == _lib.MOE_EINVAL and "overlap" in _lib.last_error()
    assert plane.launch_count == before
