"""Groups whose fp32 sums are equal or nearly so although the numbers behind them are not: large biases that lie close together.

A sigmoid's key s + bias is rounded to fp32, the sum of a group's two once more: with biases near B each rounding is up to half a
step of B, six of them between two groups, up to four steps of kmax 2^-23 in all.  The rows here are those of many random ones where
these add up, so that the definition's order is not that of the real sums."""
import numpy as np
import pytest
import torch

import npu_offload_b200 as nob
from tests.route_util import choose, keys

pytestmark = pytest.mark.gpu
E, SIZE = 32, 16
LIVE = [3, 9, 18, 27]  # the two largest of either group


def biases(rng, B):
    b = (B + rng.uniform(0, 0.1, E)).astype(np.float32)
    b[0], b[16] = B, np.float32(B) + np.float32(0.1)
    return b


def rows_of(l):
    """[n, 4] logits of the live experts as rows of E; the others' sigmoids are nothing beside a bias."""
    rows = np.full((len(l), E), -30, np.float32)
    rows[:, LIVE] = l
    return rows


def misleading(rng, B, n=1_000_000):
    """(logits, bias) of rows whose real sums lie further apart than 2.5 steps of B the other way than the definition has them."""
    b = biases(rng, B)
    l = rng.uniform(-1, 0.5, (n, 4)).astype(np.float32)
    s = 1 / (1 + np.exp(-l.astype(np.float64)).astype(np.float32))
    key = s + b[LIVE]
    assert s.dtype == key.dtype == np.float32
    score = np.stack([key[:, 0] + key[:, 1], key[:, 2] + key[:, 3]], -1)
    real = s.astype(np.float64) + b[LIVE]
    gap = real[:, 2] + real[:, 3] - real[:, 0] - real[:, 1]
    wrong = np.where(score[:, 0] >= score[:, 1], gap, -gap) / (B * 2.0 ** -23)
    return rows_of(l[wrong > 2.5]), b


def from_score(s):
    """An fp32 logit whose sigmoid, rounded as the router does, is s."""
    at = np.float32(np.log(float(s) / (1 - float(s))))
    for k in range(400):
        for l in {at + np.float32(k * 2.0 ** -26), at - np.float32(k * 2.0 ** -26)}:
            if np.float32(1) / (np.float32(1) + np.exp(-np.float64(l)).astype(np.float32)) == s:
                return np.float32(l)
    raise AssertionError(s)


def equal_sums():
    """Both groups' fp32 sums are 257.10907; the words of the second lie 411 steps above those of the first."""
    h = lambda t: np.float32(float.fromhex(t))  # noqa: E731
    b = np.full(E, 128, np.float32)
    b[16] = np.float32(128.1)
    b[LIVE] = [h("0x1.0004cap+7"), h("0x1.00217p+7"), h("0x1.001eb2p+7"), h("0x1.0020bcp+7")]
    l = [from_score(h(t)) for t in ("0x1.022fe8p-1", "0x1.0f6b04p-1", "0x1.5136p-2", "0x1.4fd2fap-1")]
    key = torch.tensor(np.array(l)), torch.tensor(b[LIVE])
    k = keys(*key, "sigmoid")
    assert k[0] + k[1] == k[2] + k[3] == np.float32(257.10907)
    return rows_of(np.array([l], np.float32)), b


def check(rows, b):
    logits, bias = torch.tensor(rows, device="cuda"), torch.tensor(b, device="cuda")
    # few tokens a call and many take different kernels, by the number of SMs
    many = 64 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    with nob.MoEDataPlane(64, 64, E, 2, n_layers=1, max_tokens=16, scoring="sigmoid") as p:
        want = choose(logits, 2, 1, 2, bias, "sigmoid")
        assert torch.equal(p.route_groups(logits, 2, 1, bias=bias)[0].cpu(), want)
        at = torch.arange(many) % len(rows)
        assert torch.equal(p.route_groups(logits[at.cuda()], 2, 1, bias=bias)[0].cpu(), want[at])
        assert p.status() == 0


def test_equal_sums_of_unequal_numbers():
    check(*equal_sums())


@pytest.mark.parametrize("B", [64, 128, 1024, 4096])
def test_sums_that_roundings_put_in_another_order(B):
    rng, found = np.random.default_rng(B), 0
    for _ in range(6):
        rows, b = misleading(rng, B)
        found += len(rows)
        if len(rows):
            check(rows, b)
    assert found or B < 1024  # (rare below)
