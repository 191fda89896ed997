"""The router's load-balance loss, its counts and its gradient against the 64-bit definition."""
import pytest
import torch

from tests.fp8_util import EPS, balance64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def planes():
    from npu_offload_b200 import MoEDataPlane
    cache = {}

    def get(E, K, scoring):
        if (E, K, scoring) not in cache:
            cache[E, K, scoring] = MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=scoring)
        return cache[E, K, scoring]
    yield get
    for p in cache.values():
        p.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(seed, T, E, K, spread=2.0):
    g = gen(seed)
    l = torch.randn(T, E, generator=g, device="cuda") * spread
    return l, l.topk(K, -1)[1].int(), g


def check(p, logits, idx, offsets, mask, scoring, grad=None):
    loss, st = p.balance_loss(logits, idx, offsets=offsets, mask=mask)
    d = p.balance_loss_backward(logits, st, grad)
    assert p.status() == 0
    want, counts, dw = balance64(logits, idx, offsets, mask, scoring, 1.0 if grad is None else float(grad))
    assert torch.equal(st.counts, counts)
    # a score is off by the difference to the maximum (its rounding is a relative error of exp), exp (2 ulp), the sum
    # of E of them and the quotient; sums of scores are all of one sign
    E, K = logits.shape[1], idx.shape[1]
    seen = torch.where(logits.isfinite(), logits, 0.0)
    score = (float(seen.max() - seen.min()) if logits.numel() else 0.0) + 16 + 40
    assert abs(float(loss) - float(want)) <= score * EPS * abs(float(want)) + 1e-30
    if logits.shape[0]:
        # sigmoid near 1: 1 - s is off by the rounding of s
        scale = (dw.abs().amax(-1, keepdim=True))
        f = st.counts.double().amax() * E / K
        n = max(1, int(st.tokens[:-1][st.tokens[:-1] > 0].min()) if bool((st.tokens[:-1] > 0).any()) else 1)
        top = (1.0 if grad is None else abs(float(grad))) * f / n / n
        assert bool(((d.double() - dw).abs() <= (2 * score + 40) * EPS * (scale + 2 * top)).all())
    return loss, st, d


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 2), (3, 60, 6), (15, 128, 8), (16, 33, 4), (17, 256, 16), (1000, 160, 8),
                                   (4099, 64, 1), (20000, 128, 8), (30011, 256, 8)])
def test_one_sequence(planes, T, E, K, scoring):
    logits, idx, g = inputs(T + E, T, E, K)
    check(planes(E, K, scoring), logits, idx, None, None, scoring, torch.tensor(0.37, device="cuda"))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cuts", [[0, 0], [0, 700], [5, 690], [0, 1, 2, 3, 700], [0, 0, 0, 700, 700], [3, 16, 17, 17, 48, 49, 640],
                                  [0, 0, 0, 0], list(range(0, 701, 7)), [700, 700]])
def test_sequences(planes, cuts, scoring):
    logits, idx, g = inputs(len(cuts), 700, 128, 8)
    off = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    mask = torch.rand(700, generator=g, device="cuda") > 0.3
    mask[17:48] = False  # a sequence of which nothing counts
    for m in (None, mask, mask.to(torch.uint8) * 255):
        _, st, d = check(planes(128, 8, scoring), logits, idx, off, m, scoring)
        assert int(st.tokens[-1]) == int((st.tokens[:-1] > 0).sum())
        assert bool((d[: cuts[0]] == 0).all()) and bool((d[cuts[-1]:] == 0).all())
        if m is not None:
            assert bool((d[~mask] == 0).all())


def test_no_sequences_of_tokens(planes):
    for off in (None, torch.zeros(4, dtype=torch.int32, device="cuda")):
        loss, st = planes(8, 2, "softmax").balance_loss(torch.zeros(0, 8, device="cuda"),
                                                        torch.zeros(0, 2, dtype=torch.int32, device="cuda"), offsets=off)
        assert float(loss) == 0 and int(st.counts.abs().sum()) == 0 and int(st.tokens.abs().sum()) == 0
        assert planes(8, 2, "softmax").balance_loss_backward(torch.zeros(0, 8, device="cuda"), st).shape == (0, 8)


def test_many_sequences(planes):
    logits, idx, g = inputs(5, 5000, 16, 2)
    cuts = torch.cat([torch.zeros(1, device="cuda"), (torch.rand(1998, generator=g, device="cuda") * 5000).sort()[0],
                      torch.full((1,), 5000.0, device="cuda")]).int()
    check(planes(16, 2, "softmax"), logits, idx, cuts, None, "softmax")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_extreme_logits_and_masked_rows_of_anything(planes, scoring):
    logits, idx, g = inputs(7, 90, 128, 8)
    logits[3, 5:] = -float("inf")
    logits[4] = torch.finfo(torch.float32).min
    logits[5] *= 30
    logits[6] = 0
    idx[10] = -1  # a token without a choice still has scores
    idx[11, 3:] = -5
    mask = torch.ones(90, dtype=torch.bool, device="cuda")
    mask[20:30] = False
    clean = check(planes(128, 8, scoring), logits, idx, None, mask, scoring)
    logits[20], logits[21], logits[22] = float("nan"), float("inf"), -float("inf")
    idx[23] = 2 ** 30
    again = planes(128, 8, scoring).balance_loss(logits, idx, mask=mask)
    d = planes(128, 8, scoring).balance_loss_backward(logits, again[1])
    assert torch.equal(again[0], clean[0]) and torch.equal(again[1].counts, clean[1].counts) and torch.equal(d, clean[2])
    assert planes(128, 8, scoring).status() == 0
    logits[0, 0] = float("nan")
    assert planes(128, 8, scoring).balance_loss(logits, idx, mask=mask)[0].isnan()


def test_the_gradient_is_the_slope_of_the_loss(planes):
    """Differences of the kernel's own loss: steps of 2^-5 in one logit, the third derivative's share left over."""
    for scoring in ("softmax", "sigmoid"):
        p = planes(8, 2, scoring)
        logits, idx, _ = inputs(3, 4, 8, 2, spread=1.0)
        _, st = p.balance_loss(logits, idx)
        d = p.balance_loss_backward(logits, st)
        h = 2.0 ** -5
        for t in range(4):
            for e in range(8):
                s = torch.zeros_like(logits)
                s[t, e] = h
                up, down = (float(p.balance_loss(logits + k * s, idx)[0]) for k in (1, -1))
                # |L'''| <= 6 sum_e f_e P_e / T for softmax or sigmoid shares (each derivative of p is at most p times a
                # number below 2); loss rounded to 64 half steps
                lim = h * h / 6 * 16 + 2 * 64 * EPS * abs(up) / (2 * h)
                assert abs((up - down) / (2 * h) - float(d[t, e])) <= lim


def test_bad_indices_and_offsets_are_reported(planes):
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    p = planes(128, 8, "softmax")
    logits, idx, _ = inputs(2, 50, 128, 8)
    bad = idx.clone()
    bad[7, 3] = 128
    _, st = p.balance_loss(logits, bad)
    assert p.status() == MOE_EINVAL and p.status() == MOE_OK
    assert int(st.counts.sum()) == 50 * 8 - 1
    for off in ([0, 30, 20, 50], [0, 51], [-1, 50], [40, 2 ** 31 - 1, 50]):
        _, st = p.balance_loss(logits, idx, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
        p.balance_loss_backward(logits, st)
        assert p.status() == MOE_EINVAL and p.status() == MOE_OK


def test_views_streams_and_graphs(planes):
    p = planes(128, 8, "softmax")
    wide, idx, g = inputs(9, 500, 256, 8)
    logits = wide[:, 100:228]  # rows apart, an odd address
    idx = logits.topk(8, -1)[1].int()
    loss, st, d = check(p, logits, idx, None, None, "softmax")
    for _ in range(3):  # nothing depends on timing
        again = p.balance_loss(logits, idx)
        assert torch.equal(again[0], loss) and torch.equal(p.balance_loss_backward(logits, again[1]), d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    l2, st2 = p.balance_loss(logits, idx, stream=s)
    d2 = p.balance_loss_backward(logits, st2, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(l2, loss) and torch.equal(d2, d)
    graph, src = torch.cuda.CUDAGraph(), torch.zeros_like(logits)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        l3, st3 = p.balance_loss(src, idx)
        d3 = p.balance_loss_backward(src, st3)
    torch.cuda.synchronize()
    src.copy_(logits)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(l3, loss) and torch.equal(d3, d) and torch.equal(st3.counts, st.counts)


def test_inside_an_autograd_function(planes):
    """The explicit pair of calls as a training program wraps it: the gradient reaches the logits' producer."""
    p = planes(8, 2, "softmax")

    class Balance(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, idx):
            loss, ctx.stats = p.balance_loss(logits.detach(), idx)
            ctx.save_for_backward(logits)
            return loss

        @staticmethod
        def backward(ctx, grad):
            (logits,) = ctx.saved_tensors
            return p.balance_loss_backward(logits.detach(), ctx.stats, grad.contiguous()), None

    g = gen(4)
    x, w = torch.randn(20, 16, generator=g, device="cuda"), torch.randn(16, 8, generator=g, device="cuda", requires_grad=True)
    idx = (x @ w).topk(2, -1)[1].int()
    (0.5 * Balance.apply(x @ w, idx)).backward()
    logits = (x @ w).detach()
    d = balance64(logits, idx, None, None, "softmax", 0.5)[2]
    want = x.double().T @ d
    # the kernel's gradient, off by less than 200 half steps of its rows' largest, through a product of 20 terms in fp32
    lim = (200 + 40) * EPS * (x.double().abs().T @ d.abs().amax(-1, keepdim=True).expand_as(d)) + 1e-12
    assert bool(((w.grad.double() - want).abs() <= lim).all())
