"""Routing limited to groups of experts, and the weights' gradient: choices equal to the definition's, numbers against 64 bits.

Tolerances (steps of 2^-24, relative; |l| <= 16, so |l - max| <= 32): a difference of logits is off by 32 of them as an
exponent, its multiplication by log2 e by 1.25 times that, the exponential by 4, the sums of the 256 values by 13 levels, each
quotient and product by 1: twice (32 + 40 + 4) + 13 + 4 = 169 < 2^-16 for a weight.  A gradient's terms are weights times
another sum of weights: two such errors and a few roundings, < 2^-14 of the terms' size."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.route_util import backward64, choose, keys, weights64

pytestmark = pytest.mark.gpu
WEIGHT, GRAD = 2.0 ** -16, 2.0 ** -14
CASES = [(8, 2, 4, 2), (8, 8, 1, 1), (16, 4, 16, 5), (33, 1, 1, 1), (32, 6, 32, 7), (60, 4, 4, 2), (60, 16, 1, 1), (64, 8, 8, 3), (96, 5, 3, 2), (120, 8, 5, 2),
         (128, 8, 8, 3), (128, 8, 1, 1), (128, 3, 4, 4), (130, 6, 13, 4), (160, 6, 8, 3), (170, 16, 17, 9), (200, 7, 1, 1), (200, 7, 25, 3), (224, 9, 7, 2),
         (248, 8, 31, 4), (255, 8, 3, 1), (256, 8, 8, 4), (256, 16, 1, 1), (256, 16, 32, 32), (256, 8, 2, 1), (250, 10, 10, 10)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def plane(E, K, scoring):
    return nob.MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=16, scoring=scoring)


def check(p, logits, groups, top, bias=None, renormalize=True, scale=1.0):
    idx, w = p.route_groups(logits, groups, top, bias=bias, renormalize=renormalize, scale=scale)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == (logits.shape[0], p.K)
    assert torch.equal(idx.cpu(), choose(logits, groups, top, p.K, bias, p.scoring))
    want = weights64(logits, idx, p.scoring, renormalize, scale)
    assert ((w.double() - want).abs() <= WEIGHT * want.abs() + 1e-37).all()
    return idx, w


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K,groups,top", CASES)
def test_choices_and_weights(E, K, groups, top, scoring):
    with plane(E, K, scoring) as p:
        g = gen(E + K)
        for T in (1, 7, 130):
            logits = (2 * torch.randn(T, E, generator=g, device="cuda")).clamp(-16, 16)
            bias = 0.3 * torch.randn(E, generator=g, device="cuda") if scoring == "sigmoid" else None
            check(p, logits, groups, top, bias)
            check(p, logits, groups, top, None, renormalize=False, scale=2.5)
        assert p.status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K,groups,top", CASES)
def test_ties_and_near_ties(E, K, groups, top, scoring):
    """Few values; values a step apart; all the same; keys that are a bias's difference; scores far below one."""
    with plane(E, K, scoring) as p:
        g = gen(2 * E + K)
        rnd = torch.randn(40, E, generator=g, device="cuda")
        step = torch.randint(0, 40, (40, E), generator=g, device="cuda")
        check(p, (rnd * 2).round() / 2, groups, top)
        check(p, torch.zeros(3, E, device="cuda"), groups, top)
        check(p, torch.zeros(3, E, device="cuda") * torch.where(rnd[:3] > 0, 1.0, -1.0), groups, top)  # 0 and -0
        check(p, 1 + step * 2.0 ** -23, groups, top)
        check(p, -1 - step * 2.0 ** -20, groups, top)
        check(p, rnd * 1e-3 - 15, groups, top)
        if scoring == "sigmoid":
            bias = -torch.sigmoid(rnd[0]) + 1e-6 * rnd[1]
            check(p, rnd[:1] + 1e-6 * rnd[2:], groups, top, bias)
            check(p, rnd, groups, top, 1e4 * rnd[3])
            check(p, rnd, groups, top, torch.where(rnd[4] > 0, 0.0, float("-inf")))
            idx = p.route_groups(rnd - 60, groups, top)[0]
            assert torch.equal(idx.cpu(), choose(rnd - 60, groups, top, K, None, scoring))
        assert p.status() == 0


@pytest.mark.parametrize("E,K,groups,top", [(16, 4, 4, 2), (128, 8, 8, 3), (256, 8, 8, 4)])
def test_many_tokens(E, K, groups, top):
    """More than a wave of warps; tokens that are done again are among them."""
    for scoring in ("softmax", "sigmoid"):
        with plane(E, K, scoring) as p:
            g = gen(E)
            logits = torch.randn(30011, E, generator=g, device="cuda")
            bias = 0.05 * torch.randn(E, generator=g, device="cuda") if scoring == "sigmoid" else None
            idx, w = p.route_groups(logits, groups, top, bias=bias)
            key = torch.from_numpy(keys(logits, bias, scoring)).cuda()
            best = key.view(-1, groups, E // groups).sort(dim=-1, descending=True)[0]
            score = best[..., 0] if scoring == "softmax" else best[..., 0] + best[..., 1]
            chosen = score.sort(dim=-1, descending=True, stable=True)[1][:, :top]
            mask = torch.zeros_like(score, dtype=torch.bool).scatter(1, chosen, True).repeat_interleave(E // groups, 1)
            want = torch.where(mask, key, float("-inf")).sort(dim=-1, descending=True, stable=True)[1][:, :K]
            assert torch.equal(idx.long(), want)
            exact = weights64(logits, idx, scoring, True, 1.0)
            assert ((w.double() - exact).abs() <= WEIGHT * exact).all() and p.status() == 0


def test_one_group_is_the_plain_router():
    for scoring in ("softmax", "sigmoid"):
        with plane(128, 8, scoring) as p:
            g = gen(3)
            logits, bias = torch.randn(500, 128, generator=g, device="cuda"), None if scoring == "softmax" else 0.1 * torch.randn(128, generator=g, device="cuda")
            a, b = p.route_groups(logits, 1, 1, bias=bias), p.route_topk(logits, bias)
            assert torch.equal(a[0], b[0]) and (a[1] - b[1]).abs().max() <= 2 * WEIGHT


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_experts(scoring):
    """-inf logits: a softmax gives them nothing, and they come last; a row of nothing else is an error."""
    from npu_offload_b200._lib import MOE_ENONFINITE, MOE_OK
    with plane(32, 6, scoring) as p:
        g = gen(5)
        logits = torch.randn(64, 32, generator=g, device="cuda")
        for t in range(64):
            logits[t, torch.randperm(32, generator=g, device="cuda")[: t // 2]] = float("-inf")
        logits[20] = torch.finfo(torch.float32).min  # the type's lowest value masks by hand
        idx, w = p.route_groups(logits, 4, 2)
        assert torch.equal(idx.cpu(), choose(logits, 4, 2, 6, None, scoring)) and p.status() == MOE_OK
        want = weights64(logits, idx, scoring, True, 1.0)
        assert ((w.double() - want).abs() <= WEIGHT * want + 1e-37).all()
        if scoring == "softmax":
            logits[9] = float("-inf")
            idx, w = p.route_groups(logits, 4, 2)
            assert p.status() == MOE_ENONFINITE and p.status() == MOE_OK
            keep = torch.arange(64, device="cuda") != 9
            assert w[9].isnan().all() and w[keep].isfinite().all() and idx[9].tolist() == [0, 1, 2, 3, 4, 5]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_nan_is_reported_and_stays_in_its_row(scoring):
    from npu_offload_b200._lib import MOE_ENONFINITE, MOE_OK
    with plane(64, 4, scoring) as p:
        logits = torch.randn(50, 64, generator=gen(6), device="cuda")
        want = p.route_groups(logits, 8, 3)
        logits[7, 5] = float("nan")
        if scoring == "softmax":
            logits[30, 60] = float("inf")
        idx, w = p.route_groups(logits, 8, 3)
        assert p.status() == MOE_ENONFINITE and p.status() == MOE_OK
        bad = torch.zeros(50, dtype=torch.bool, device="cuda")
        bad[7], bad[30] = True, scoring == "softmax"
        assert torch.equal(idx[~bad], want[0][~bad]) and torch.equal(w[~bad], want[1][~bad]) and w[bad].isnan().all()
        assert all(len(set(r)) == 4 and min(r) >= 0 and max(r) < 64 for r in idx.tolist())
        assert torch.equal(idx.cpu(), choose(logits, 8, 3, 4, None, scoring))


def near(got, want, size):
    assert ((got.double() - want).abs() <= GRAD * size + 1e-37).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (False, 2.5)])
@pytest.mark.parametrize("E,K", [(8, 8), (16, 1), (31, 3), (60, 6), (64, 4), (100, 2), (128, 8), (160, 6), (255, 16), (256, 8)])
def test_backward(E, K, scoring, renormalize, scale):
    with plane(E, K, scoring) as p:
        g = gen(E * K)
        for T in (1, 5, 300):
            logits = (3 * torch.randn(T, E, generator=g, device="cuda")).clamp(-16, 16)
            idx = logits.topk(K, -1)[1].int()
            dw = torch.randn(T, K, generator=g, device="cuda")
            want, size = backward64(logits, idx, dw, scoring, renormalize, scale)
            got = p.route_backward(logits, idx, dw, renormalize=renormalize, scale=scale)
            near(got, want, size)
            if renormalize or scoring == "sigmoid":  # the others have none
                others = torch.ones(T, E, dtype=torch.bool, device="cuda").scatter(1, idx.long(), False)
                assert (got[others] == 0).all()
            start = torch.randn(T, E, generator=g, device="cuda")
            out = start.clone()
            p.route_backward(logits, idx, dw, renormalize=renormalize, scale=scale, out=out, accumulate=True)
            assert torch.equal(out, start + got)
            out.fill_(float("nan"))
            p.route_backward(logits, idx, dw, renormalize=renormalize, scale=scale, out=out)
            assert torch.equal(out, got)
        assert p.status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_backward_of_dropped_repeated_and_bad_choices(scoring, renormalize):
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    with plane(40, 4, scoring) as p:
        g = gen(12)
        logits, dw = torch.randn(60, 40, generator=g, device="cuda"), torch.randn(60, 4, generator=g, device="cuda")
        idx = torch.randint(-1, 40, (60, 4), generator=g, device="cuda").int()
        idx[0] = -1
        idx[1] = torch.tensor([5, 5, 5, 5])
        idx[2] = torch.tensor([-3, 7, 7, -1])
        dw[2, 0] = float("nan")  # of no choice: it reaches nothing
        want, size = backward64(logits, idx, dw, scoring, renormalize, 1.5)
        got = p.route_backward(logits, idx, dw, renormalize=renormalize, scale=1.5)
        near(got, want, size)
        assert (got[0] == 0).all() and p.status() == MOE_OK
        assert torch.equal(p.route_backward(logits, idx, dw, renormalize=renormalize, scale=1.5), got)
        worse = idx.clone()
        worse[idx < 0] = 40
        worse[0, 1] = 2 ** 31 - 1
        again = p.route_backward(logits, worse, dw, renormalize=renormalize, scale=1.5)
        assert p.status() == MOE_EINVAL and p.status() == MOE_OK and torch.equal(again, got)


def test_router_and_balance_gradients_on_one_tensor():
    """What a training step does with them, against the sum of both gradients in 64 bits."""
    from tests.fp8_util import balance64
    with plane(60, 4, "sigmoid") as p:
        g = gen(13)
        logits, dw = torch.randn(700, 60, generator=g, device="cuda"), torch.randn(700, 4, generator=g, device="cuda")
        idx, w = p.route_groups(logits, 4, 2, scale=2.5)
        loss, stats = p.balance_loss(logits, idx)
        grad = torch.full((), 0.5, device="cuda")
        d = p.balance_loss_backward(logits, stats, grad)
        before = d.clone()
        p.route_backward(logits, idx, dw, scale=2.5, out=d, accumulate=True)
        alone = p.route_backward(logits, idx, dw, scale=2.5)
        near(alone, *backward64(logits, idx, dw, "sigmoid", True, 2.5))
        assert torch.equal(d, before + alone)
        # the balance gradient is a difference of f and its mean, each of size f: off by a few steps of both, not of itself
        b = 0.5 * balance64(logits.double().cpu(), idx.cpu(), torch.tensor([0, 700]), None, "sigmoid")[2].cuda()
        s = torch.sigmoid(logits.double())
        f = stats.counts[0].double() * 60 / (4 * 700)
        size = 0.5 / 700 * s * (1 - s) / s.sum(-1, keepdim=True) * (f + (f * s / s.sum(-1, keepdim=True)).sum(-1, keepdim=True))
        assert ((before.double() - b).abs() <= 2.0 ** -18 * size).all()


def test_no_tokens_strides_streams_and_graphs():
    with plane(128, 8, "sigmoid") as p:
        assert p.route_groups(torch.zeros(0, 128, device="cuda"), 8, 3)[0].shape == (0, 8)
        assert p.route_backward(torch.zeros(0, 128, device="cuda"), torch.zeros(0, 8, device="cuda", dtype=torch.int32), torch.zeros(0, 8, device="cuda")).shape == (0, 128)
        g = gen(14)
        wide = torch.randn(99, 256, generator=g, device="cuda")
        check(p, wide[:, ::2], 8, 3)
        check(p, wide.view(-1)[1:1 + 90 * 128].view(90, 128), 8, 3)  # not at a 16-byte boundary
        data = [(torch.randn(77, 128, generator=g, device="cuda"), torch.randn(77, 8, generator=g, device="cuda")) for _ in range(2)]

        def step(logits, dw, stream=None):
            idx, w = p.route_groups(logits, 8, 3, scale=2.5, stream=stream)
            return idx, w, p.route_backward(logits, idx, dw, scale=2.5, stream=stream)

        want = [step(*d) for d in data]
        torch.cuda.synchronize()
        other = step(*data[0], stream=torch.cuda.Stream())
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
                    o[0].zero_(), o[2].zero_()
                    graph.replay()
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, v))


def test_the_library_refuses():
    from npu_offload_b200 import _lib
    L, t = nob.lib(), torch.zeros(4, 16, device="cuda")
    idx, w0 = torch.zeros(4, 4, device="cuda", dtype=torch.int32), torch.zeros(4, 4, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        with plane(16, 4, scoring) as p:
            def call(T=4, lg=t.data_ptr(), bias=None, groups=4, top=2, scale=1.0, i=idx.data_ptr(), w=w0.data_ptr(), flags=0):
                return L.moe_route_groups(p.handle, T, lg, bias, groups, top, 1, scale, i, w, flags, None)

            for kw, needle in ((dict(T=-1), "T="), (dict(T=1 << 25), "T="), (dict(groups=0), "groups"), (dict(groups=3), "divisor"), (dict(groups=33), "divisor"),
                               (dict(top=0), "top_groups"), (dict(top=5), "top_groups"), (dict(groups=16, top=3), "choices"), (dict(scale=float("nan")), "scale"),
                               (dict(lg=None), "null"), (dict(i=None), "null"), (dict(flags=2), "flag"), (dict(w=idx.data_ptr()), "overlaps"),
                               (dict(lg=t.data_ptr() + 2), "4-byte"), (dict(w=t.data_ptr()), "overlaps")):
                assert call(**kw) == _lib.MOE_EINVAL and needle in _lib.last_error(), kw
            if scoring == "softmax":
                assert call(bias=t.data_ptr()) == _lib.MOE_EINVAL and "bias" in _lib.last_error()
            z = torch.zeros(4, 16, device="cuda")

            def back(T=4, out=z.data_ptr(), scale=1.0, flags=0):
                return L.moe_route_backward(p.handle, T, t.data_ptr(), idx.data_ptr(), t.data_ptr(), 1, scale, out, flags, None)

            for kw, needle in ((dict(T=-1), "T="), (dict(out=None), "null"), (dict(out=t.data_ptr()), "overlaps"), (dict(scale=float("inf")), "scale"),
                               (dict(flags=1), "device pointers")):
                assert back(**kw) == _lib.MOE_EINVAL and needle in _lib.last_error(), kw
            assert p.launch_count == 0


# ---------------------------------------------------------------- calls of many tokens (another kernel, by size)

def sorted_choice(logits, groups, top, K, bias, scoring):
    """choose() by stable sorts on the GPU, for many tokens (NaN as -inf)."""
    key = torch.from_numpy(keys(logits, bias, scoring)).cuda()
    key = torch.where(key.isnan(), float("-inf"), key)
    T, E = key.shape
    best = key.view(T, groups, E // groups).sort(dim=-1, descending=True)[0]
    score = best[..., 0] if scoring == "softmax" or E == groups else best[..., 0] + best[..., 1]
    score = torch.where(score.isnan(), float("-inf"), score)
    chosen = score.sort(dim=-1, descending=True, stable=True)[1][:, :top]
    open_ = torch.zeros_like(score, dtype=torch.bool).scatter(1, chosen, True).repeat_interleave(E // groups, 1)
    first = open_.float().sort(dim=-1, descending=True, stable=True)[1]  # open experts in front, in order
    inside = key.gather(1, first)[:, : top * (E // groups)]
    return first.gather(1, inside.sort(dim=-1, descending=True, stable=True)[1])[:, :K].int()


MANY = [(32, 2, 8, 3), (32, 8, 1, 1), (64, 6, 8, 2), (64, 8, 4, 4), (96, 4, 4, 1), (128, 8, 8, 3), (128, 1, 2, 1), (160, 6, 8, 3), (192, 8, 2, 1), (224, 5, 8, 8),
        (256, 8, 8, 4), (256, 8, 1, 1), (256, 8, 4, 2), (256, 8, 8, 1), (256, 9, 8, 4), (248, 8, 8, 4), (240, 8, 16, 4)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K,groups,top", MANY)
def test_many_tokens_of_all_kinds(E, K, groups, top, scoring):
    """Random logits, few values, values a step apart, biases that decide, masked experts; numbers of tokens that leave a rest."""
    with plane(E, K, scoring) as p:
        g = gen(7 * E + K)
        for T in (9602, 9475):
            rnd = torch.randn(T, E, generator=g, device="cuda")
            kinds = [rnd, (rnd * 2).round() / 2, 1 + torch.randint(0, 9, (T, E), generator=g, device="cuda") * 2.0 ** -23, rnd * 1e-3 - 15]
            if scoring == "softmax":
                kinds.append(torch.where(rnd > 1, float("-inf"), rnd))
            for logits in kinds:
                bias = 0.05 * torch.randn(E, generator=g, device="cuda") if scoring == "sigmoid" else None
                for b in ({None} if bias is None else {None, bias, 1e4 * bias, torch.where(bias > 0.05, float("-inf"), bias)}):
                    for renormalize in (True, False):
                        idx, w = p.route_groups(logits, groups, top, bias=b, renormalize=renormalize, scale=1.5)
                        assert torch.equal(idx, sorted_choice(logits, groups, top, K, b, scoring))
                        want = weights64(logits, idx, scoring, renormalize, 1.5)
                        assert ((w.double() - want).abs() <= WEIGHT * want + 1e-37).all()
        assert p.status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_many_tokens_with_errors_among_them(scoring):
    from npu_offload_b200._lib import MOE_ENONFINITE, MOE_OK
    with plane(128, 8, scoring) as p:
        T = 9503
        logits = torch.randn(T, 128, generator=gen(21), device="cuda")
        want = p.route_groups(logits, 8, 3)
        bad = torch.zeros(T, dtype=torch.bool, device="cuda")
        for t in (0, 5, 1502, T - 1):
            logits[t, (t * 7) % 128] = float("nan")
            bad[t] = True
        if scoring == "softmax":
            logits[9] = float("-inf")
            logits[10, 3] = float("inf")
            bad[9] = bad[10] = True
        idx, w = p.route_groups(logits, 8, 3)
        assert p.status() == MOE_ENONFINITE and p.status() == MOE_OK
        assert torch.equal(idx[~bad], want[0][~bad]) and torch.equal(w[~bad], want[1][~bad]) and w[bad].isnan().all()
        assert torch.equal(idx, sorted_choice(logits, 8, 3, 8, None, scoring))
        if scoring == "sigmoid":
            logits = torch.randn(T, 128, generator=gen(22), device="cuda")
            bias = torch.zeros(128, device="cuda")
            bias[17] = float("nan")
            w = p.route_groups(logits, 8, 3, bias=bias)[1]
            assert p.status() == MOE_ENONFINITE and w.isnan().all()


def test_few_and_many_tokens_agree():
    """The same rows in a call of few and in one of many: the same choices and weights to the last steps."""
    for scoring in ("softmax", "sigmoid"):
        with plane(256, 8, scoring) as p:
            logits = torch.randn(10000, 256, generator=gen(23), device="cuda")
            many = p.route_groups(logits, 8, 4)
            few = p.route_groups(logits[:100].clone(), 8, 4)
            assert torch.equal(many[0][:100], few[0]) and (many[1][:100] - few[1]).abs().max() <= WEIGHT
