"""Adapters where values end: infinities beside padded ranks, in B, sums near the largest number; base alone bit for bit; calls of
few and of many tokens alike."""
import pytest
import torch

import npu_offload_b200 as nob

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


@pytest.fixture(scope="module")
def plane():
    with nob.MoEDataPlane(256, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        yield p


def make(seed, T, K, N, r, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ids = torch.randint(-1, n, (T,), generator=g, device="cuda")
    ids[:4] = torch.tensor([0, n - 1, 0, -1], device="cuda")
    return dict(base=f(T, N).to(dtype), x=f(T, K).to(BF), a=(f(n, r, K) * K ** -0.5).to(BF), b=(f(n, N, r) * r ** -0.5).to(BF), ids=ids.to(torch.int32),
                scale=0.5 + torch.rand(n, generator=g, device="cuda"))


def definition(base, x, a, b, ids, scale):
    out = base.double()
    for t, i in enumerate(ids.tolist()):
        if i >= 0:
            out[t] += (float(scale[i]) * (a[i].double() @ x[t].double())) @ b[i].double().T
    return out


def same_ends(got, want):
    """NaN where the definition has it, infinities of its signs; other values finite."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.where(got.isinf(), got, 0).double(), torch.where(want.isinf(), want, 0))


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("r", [8, 24, 40, 56, 72, 120, 16, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinities_in_x(plane, T, r, dtype):
    """All of A and B of one sign: every inner sum is the infinity of x's sign, and so is every result of that token."""
    m = make(r, T, 136, 77, r, 3, dtype)
    m["a"][0], m["b"][0] = m["a"][0].abs() + 0.01, m["b"][0].abs() + 0.01
    clean = plane.add_lora(**m)
    m["x"][0, 100], m["x"][2, 3] = INF, -INF
    got, want = plane.add_lora(**m), definition(**m)
    assert (want[0] == INF).all() and (want[2] == -INF).all()
    same_ends(got, want)
    assert torch.equal(got[3:], clean[3:]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("r", [24, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scales_that_are_no_numbers(plane, T, r, dtype):
    m = make(r, T, 136, 77, r, 3, dtype)
    m["a"][0], m["b"][0], m["x"] = m["a"][0].abs() + 0.01, m["b"][0].abs() + 0.01, m["x"].abs() + 0.01
    m["scale"][0], m["scale"][2] = INF, float("nan")
    same_ends(plane.add_lora(**m), definition(**m))
