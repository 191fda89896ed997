"""How exact the balance loss's scores and gradients are where fp32 decides: far and saturated logits.

Bounds are counted in half steps of fp32 (EPS, relative): the hardware's 2^x is off by 2 ulp (4 half steps) at most, each
rounded operation by one.  The sigmoid's exp(d) = 2^t (1 + r) is off by 5, its last operation being a fused one; the
softmax's 2^(d log2 e) by 4 and, for the rounded exponent, 1.25 |d|.
"""
import pytest
import torch

from tests.fp8_util import EPS

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["softmax", "sigmoid"])
def plane(request):
    from npu_offload_b200 import MoEDataPlane
    cache = {}

    def get(E, K=1):
        if (E, K) not in cache:
            cache[E, K] = MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=request.param)
        return cache[E, K]
    yield get
    for p in cache.values():
        p.close()


def scores64(logits, scoring):
    l = logits.double()
    if scoring == "softmax":
        return torch.softmax(l, -1)
    s = torch.sigmoid(l)
    return s / (s.sum(-1, keepdim=True) + 1e-20)


@pytest.mark.parametrize("E", [8, 7])
def test_a_score_is_off_by_a_few_half_steps(plane, E):
    """One token with one choice: the loss is E times that expert's score.

    Logits are multiples of 2^-10 below 64, so that their difference d to the largest is exact.  Softmax: the score's
    exp 4 + 1.25 |d| half steps, and so those of the sum, weighed by their share (e^-d 1.25 d is below 1/2: 7 of them below
    4).  Sigmoid x / (1 + x): x 5, 1 + x, the quotient and the product one each: 8.  The sum of eight adds 4 roundings,
    1e-20 one and one of its own, its inverse one, the score's product one, the loss's conversion one: 9."""
    p = plane(E)
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = torch.round(torch.randn(400, E, generator=g, device="cuda").clamp(-4, 4) * 12 * 1024) / 1024
    logits[200:] -= logits[200:].amax(-1, keepdim=True)  # none above 0
    idx = logits.argmin(-1, keepdim=True).int()
    want = E * scores64(logits, p.scoring).gather(1, idx.long())[:, 0]
    got = torch.stack([p.balance_loss(logits[t:t + 1], idx[t:t + 1])[0] for t in range(400)]).double()
    assert p.status() == 0
    off = (got - want).abs() / want / EPS
    span = (logits.amax(-1) - logits.amin(-1)).double()
    limit = 4 + 1.25 * span + (4 + 4) + 9 if p.scoring == "softmax" else 8 + 8 + 9
    assert bool((off <= limit).all()), float((off - limit).max())


@pytest.mark.parametrize("low,high", [(12.0, 20.0), (-20.0, 20.0), (60.0, 80.0), (-2.0, 2.0)])
@pytest.mark.parametrize("E,K", [(128, 8), (60, 4)])
def test_gradients_of_saturated_scores(plane, E, K, low, high):
    """1 - s of a sigmoid near 1 is as exact as s: each gradient against its own slope p (softmax) or s (1 - s) / S.

    Half steps: s 8, 1 - s 8, their product one; S 8 for its terms, 14 for the sum (8 values a lane, then 5 steps, 1e-20);
    its inverse and the product with it one each: 41 for the slope (softmax 4 + 1.25 |d| and 1 |d| for d itself, twice, and
    16).  f: three.  f . p: 8 and 14 for the sum, 32 for p: 54.  Their difference one.  Below
    2^-126 numbers are 2^-149 apart: two roundings of the slope and one of the gradient, of half that each."""
    p = plane(E, K)
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = low + (high - low) * torch.rand(300, E, generator=g, device="cuda")
    idx = logits.topk(K, -1)[1].int()
    _, st = p.balance_loss(logits, idx)
    d = p.balance_loss_backward(logits, st).double()
    l = logits.double()
    f = st.counts.double()[0] * E / (K * 300) / 300
    pr = scores64(logits, p.scoring)
    slope, far = pr, 2.25 * 2 * (l.amax(-1, keepdim=True) - l.amin(-1, keepdim=True))
    if p.scoring == "sigmoid":
        slope, far = torch.sigmoid(-l) * pr, 0.0
    inner = (f * pr).sum(-1, keepdim=True)
    limit = EPS * slope * ((42 + far) * (f - inner).abs() + 3 * f + (55 + far) * inner) + 1.5 * 2.0 ** -149
    off = (d - slope * (f - inner)).abs()
    assert bool((off <= limit).all()), float((off / limit).max())
    assert p.status() == 0
