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


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("r,N", [(8, 77), (16, 64), (24, 136), (64, 264), (128, 33)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinities_in_b(plane, T, r, N, dtype):
    """A finite inner sum times an infinity is one, whatever the inner sum is held in."""
    m = make(r + N, T, 136, N, r, 3, dtype)
    for n in range(0, N, 5):
        m["b"][0, n, n % r] = INF if n % 2 else -INF
    m["b"][0, 11, :] = INF  # of both signs among the products: NaN
    m["x"][2] = 0  # 0 times an infinity
    clean = plane.add_lora(**{**m, "b": torch.where(m["b"].isinf(), 0, m["b"])})
    got, want = plane.add_lora(**m), definition(**m)
    assert want[0].isinf().any() and want[2].isnan().any()
    same_ends(got, want)
    plain = [n for n in range(N) if n % 5 and n != 11]
    assert torch.equal(got[:, plain], clean[:, plain])  # columns without one
    others = m["ids"] != 0
    assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_inner_sums_beyond_the_largest_bf16(plane, T, dtype):
    """Inner sums of 2^127 (2 - 2^-9), which bf16 rounds to an infinity; the result is 4 - 2^-8 beside a base of 0."""
    m = make(1, T, 64, 40, 16, 2, dtype)
    m["ids"].zero_()
    m["base"].zero_(), m["x"].zero_(), m["a"].zero_(), m["b"].zero_()
    m["x"][:, 0], m["x"][:, 1], m["a"][0, 3, :2], m["b"][0, :, 3], m["scale"][0] = 2.0 ** 127, 2.0 ** 119, 1.0, 2.0 ** -126, 1.0
    m["a"][0, 3, 0], m["a"][0, 3, 1] = 2 - 2.0 ** -7, 1.5
    want = definition(**m)
    got = plane.add_lora(**m)
    assert want[0, 0] == 2 * (2 - 2.0 ** -9)
    # off by half a step of the result, and by 2^-16 of the sum where that is held in two parts
    assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + (2.0 ** -16 if dtype == BF else 2.0 ** -23)) * want).all()


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("N", [64, 77])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_base_alone_keeps_its_zeros(plane, T, N, dtype):
    """Zeros of either sign and NaN among the tokens without an adapter."""
    m = make(N, T, 72, N, 16, 3, dtype)
    m["ids"][1::2] = -1
    m["base"][:, ::3] = -0.0
    m["base"][:, 1::7] = float("nan")
    none, bits = m["ids"] < 0, torch.int16 if dtype == BF else torch.int32
    out, base = plane.add_lora(**m)[none], m["base"][none]
    assert torch.equal(out.isnan(), base.isnan())
    assert torch.equal(torch.where(base.isnan(), 0, out).view(bits), torch.where(base.isnan(), 0, base).view(bits))


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("r", [16, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_what_is_left_where_base_and_adapter_cancel(plane, T, r, dtype):
    """fp32 sums (steps of 2^-24 of the sizes, as the other tests of this call count them), and for bf16 results of many tokens the inner
    sums to 2^-16 of each: nothing of the size of a bf16 step of base reaches the result."""
    m = make(r, T, 512, 96, r, 2, dtype)
    m["ids"].clamp_(min=0)
    m["base"].zero_()
    m["base"] = (-definition(**m)).to(dtype)
    got, want = plane.add_lora(**m), definition(**m)
    i = m["ids"].long()
    low = torch.einsum("t,tk,trk->tr", m["scale"][i].double(), m["x"].double(), m["a"][i].double()).abs()
    size = torch.einsum("t,tk,trk,tnr->tn", m["scale"][i].double(), m["x"].double().abs(), m["a"][i].double().abs(), m["b"][i].double().abs())
    held = torch.einsum("tr,tnr->tn", low, m["b"][i].double().abs())
    bound = torch.finfo(dtype).eps / 2 * want.abs() + (512 / 128 + r + 40) * 2.0 ** -24 * (size + m["base"].double().abs())
    if dtype == BF and T == 150:
        bound += 2.0 ** -16 * held
    assert ((got.double() - want).abs() <= bound).all()
