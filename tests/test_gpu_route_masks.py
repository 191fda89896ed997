"""Masked experts: by logits of -inf under softmax scoring, by biases under sigmoid; what a logit of -inf is with a bias; in calls of
few tokens and of many, which take different kernels by the number of SMs."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.route_util import choose, weights64

pytestmark = pytest.mark.gpu
WEIGHT = 2.0 ** -16  # (as the other tests of this call derive it)


def plane(E, K, scoring):
    return nob.MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=scoring)


def check(p, logits, groups, top, bias=None):
    many = 64 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    want = choose(logits, groups, top, p.K, bias, p.scoring)
    for at in (torch.arange(len(logits)), torch.arange(many) % len(logits)):
        idx, w = p.route_groups(logits[at.cuda()], groups, top, bias=bias)
        assert torch.equal(idx.cpu(), want[at])
        exact = weights64(logits[at.cuda()], idx, p.scoring, True, 1.0)
        assert ((w.double() - exact).abs() <= WEIGHT * exact + 1e-37).all()
    assert p.status() == 0
    return want


@pytest.mark.parametrize("E,K,groups,top", [(32, 4, 4, 2), (128, 8, 8, 3), (256, 8, 8, 4), (256, 8, 1, 1)])
def test_sigmoid_masks_by_bias(E, K, groups, top):
    g = torch.Generator(device="cuda").manual_seed(E)
    logits, bias = torch.randn(60, E, generator=g, device="cuda"), 0.1 * torch.randn(E, generator=g, device="cuda")
    masked = torch.randperm(E, generator=g, device="cuda")[: E // 4]
    with plane(E, K, "sigmoid") as p:
        for value in (float("-inf"), -10.0):  # -inf, or far below all others
            b = bias.clone()
            b[masked] = value
            assert not torch.isin(check(p, logits, groups, top, b), masked.cpu().int()).any()


def test_sigmoid_of_a_logit_of_minus_infinity_has_its_bias_for_a_key():
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, bias = torch.randn(50, 32, generator=g, device="cuda"), torch.zeros(32, device="cuda")
    logits[:, 5], logits[:, 20] = float("-inf"), float("-inf")
    bias[5], bias[20] = 2.0, -2.0
    with plane(32, 4, "sigmoid") as p:
        want = check(p, logits, 1, 1, bias)
        assert (want[:, 0] == 5).all() and not (want == 20).any()  # the best of all, by its bias, with a weight of 0
        idx, w = p.route_groups(logits, 1, 1, bias=bias)
        assert (w[:, 0] == 0).all()
        nothing = torch.full((1, 32), float("-inf"), device="cuda")  # weights of 0, and no error
        assert check(p, nothing, 4, 2, bias)[0, 0] == 5
        assert (p.route_groups(nothing, 4, 2, bias=bias)[1] == 0).all()


@pytest.mark.parametrize("E,K,groups,top", [(32, 4, 4, 2), (256, 8, 8, 4)])
def test_softmax_masks_by_logits(E, K, groups, top):
    g = torch.Generator(device="cuda").manual_seed(E + 1)
    logits = torch.randn(60, E, generator=g, device="cuda")
    logits[torch.rand(60, E, generator=g, device="cuda") < 0.6] = float("-inf")
    logits[:, 1] = 0
    with plane(E, K, "softmax") as p:
        check(p, logits, groups, top)
