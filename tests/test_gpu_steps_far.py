"""Tensors of more than 2^31 values: the norm, grouped routing and adapters at their last rows, against calls on those rows alone."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.norm_util import norm_backward64

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
LAST = 300


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 60 GB")
    yield
    torch.cuda.empty_cache()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("C", [16384, 4099])
def test_norm(C):
    T = 2 ** 31 // C + 2 * LAST
    with nob.MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        x = torch.empty(T, C, device="cuda", dtype=BF).normal_(generator=gen(1))
        r = torch.empty(T, C, device="cuda", dtype=BF).normal_(generator=gen(2))
        w = 1 + 0.2 * torch.randn(C, generator=gen(3), device="cuda")
        n = p.add_norm(x, w, r, fp8=C % 16 == 0)
        few = p.add_norm(x[-LAST:].clone(), w, r[-LAST:].clone(), fp8=C % 16 == 0)
        assert same(n.sum[-LAST:], few.sum)
        # a call of few rows adds up a row's squares in another order: rstd is off by 2^-19 at most, and so is y before its rounding
        assert ((n.rstd[-LAST:] - few.rstd).abs() <= 2.0 ** -18 * few.rstd).all()
        assert ((n.y[-LAST:].double() - few.y.double()).abs() <= (2.0 ** -7 + 2.0 ** -18) * few.y.double().abs()).all()
        if C % 16 == 0:
            assert same(n.fp8.scale[-LAST:], few.fp8.scale)
        dx, dw = p.add_norm_backward(x, n.sum, w, n.rstd, dsum=r, weight_grad=False)
        # as the gradient's other tests derive it: half a step, and a few of the terms' size
        rows = slice(T - LAST, T)
        want, _, size, _ = norm_backward64(x[rows], n.sum[rows], w, n.rstd[rows], r[rows])
        assert dw is None and ((dx[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size + 1e-40).all()
        if C % 8 == 0:  # (in other rows, how values fall to threads depends on where a row begins)
            small, _ = p.add_norm_backward(x[rows].clone(), few.sum, w, n.rstd[rows].clone(), dsum=r[rows].clone(), weight_grad=False)
            assert same(dx[rows], small)
        assert p.status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing_and_its_gradient(scoring):
    T, E, K = 2 ** 31 // 256 + 2 * LAST, 256, 8
    with nob.MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=scoring) as p:
        logits = torch.empty(T, E, device="cuda").normal_(generator=gen(4))
        few = logits[-LAST:].clone()
        for renormalize in (True, False):
            idx, w = p.route_groups(logits, 8, 4, renormalize=renormalize)
            want, weight = p.route_groups(few, 8, 4, renormalize=renormalize)
            assert torch.equal(idx[-LAST:], want) and ((w[-LAST:] - weight).abs() <= 2.0 ** -15 * weight).all()
            d = p.route_backward(logits, idx, w, renormalize=renormalize)
            assert same(d[-LAST:], p.route_backward(few, want, w[-LAST:].clone(), renormalize=renormalize))
            assert same(d[:LAST], p.route_backward(logits[:LAST].clone(), idx[:LAST].clone(), w[:LAST].clone(), renormalize=renormalize))
            del d
        assert p.status() == 0


@pytest.mark.parametrize("N,dtype", [(2080, BF), (2083, F32)])
def test_adapters(N, dtype):
    T, K, r, n = 1 << 20, 64, 16, 4096
    with nob.MoEDataPlane(64, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        base = torch.empty(T, N, device="cuda", dtype=dtype).normal_(generator=gen(5))
        x = torch.empty(T, K, device="cuda", dtype=BF).normal_(generator=gen(6))
        a, b = torch.randn(n, r, K, generator=gen(7), device="cuda").to(BF), torch.randn(n, N, r, generator=gen(8), device="cuda").to(BF)
        ids = torch.randint(-1, n, (T,), generator=gen(9), device="cuda", dtype=torch.int32)
        out = p.add_lora(base, x, a, b, ids)
        for part in (slice(T - LAST, T), slice(0, LAST)):
            want = p.add_lora(base[part].clone(), x[part].clone(), a, b, ids[part].clone())
            assert same(out[part], want)  # (a token's sums do not depend on its place)
        assert p.status() == 0
