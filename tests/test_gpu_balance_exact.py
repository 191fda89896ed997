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
