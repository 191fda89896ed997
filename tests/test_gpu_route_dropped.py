"""The gradient of routing weights at tokens without a choice: zero, whatever their logits hold."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.route_util import backward64

pytestmark = pytest.mark.gpu
ROWS = {0: "-inf", 3: "nan", 7: "inf", 8: "nan"}  # tokens without a choice, and what all of their logits are


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E,K", [(16, 2), (40, 4), (100, 9), (256, 8)])
@pytest.mark.parametrize("none", ["negative", "out of range"])
def test_tokens_without_a_choice(E, K, scoring, renormalize, none):
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    with nob.MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=scoring) as p:
        g = torch.Generator(device="cuda").manual_seed(E + K)
        logits, dw = torch.randn(11, E, generator=g, device="cuda"), torch.randn(11, K, generator=g, device="cuda")
        idx = logits.topk(K, -1)[1].int()
        idx[5, 0] = -1  # one choice of several
        empty = torch.tensor(list(ROWS), device="cuda")
        idx[empty] = -1 if none == "negative" else E
        want, size = backward64(logits, torch.where(idx < E, idx, -1), dw, scoring, renormalize, 1.5)
        for t, v in ROWS.items():
            logits[t] = float(v)
        logits[8, 3:] = 1.0  # some of them alone
        got = p.route_backward(logits, idx, dw, renormalize=renormalize, scale=1.5)
        assert (got[empty] == 0).all()
        assert ((got.double() - want).abs() <= 2.0 ** -14 * size + 1e-37).all()  # (as the other tests of this call derive it)
        start = torch.randn(11, E, generator=g, device="cuda")
        start[3, 2] = -0.0
        out = start.clone()
        p.route_backward(logits, idx, dw, renormalize=renormalize, scale=1.5, out=out, accumulate=True)
        assert torch.equal(out[empty].view(torch.int32), start[empty].view(torch.int32))  # left as it was
        assert torch.equal(out, start + got)
        assert p.status() == (MOE_OK if none == "negative" else MOE_EINVAL)
