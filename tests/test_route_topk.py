"""The router alone on the device (route_topk): refusals, sizes, and calls that overlap on the GPU."""
import pytest
import torch

import npu_offload_b200 as nob
from npu_offload_b200._lib import MoEError


@pytest.fixture
def plane(monkeypatch):
    """A plane of the host's memory whose C calls get a null context."""
    p = object.__new__(nob.MoEDataPlane)
    p.H, p.F, p.E, p.K, p._h, p._index, p._plane = 256, 64, 8, 2, None, 0, None
    p.device = torch.device("cpu")
    from npu_offload_b200 import moe
    monkeypatch.setattr(moe, "_raw_stream", lambda index: 0)
    return p


@pytest.mark.parametrize("shape", [(7,), (9,), (1,), (0,), (8, 8), ()])
def test_a_bias_of_another_size_is_refused(plane, shape):
    """A shorter one would be read behind its end."""
    with pytest.raises(ValueError, match="bias is"):
        plane.route_topk(torch.zeros(3, 8), bias=torch.zeros(shape))


@pytest.mark.parametrize("shape", [(7,), (9,), (0,), (8, 8)])
def test_route_and_set_bias_refuse_it_too(plane, shape):
    with pytest.raises(ValueError, match="bias is"):
        plane.route(torch.zeros(3, 8), bias=torch.zeros(shape))
    with pytest.raises(ValueError, match="bias is"):
        plane.set_bias(0, torch.zeros(shape))


def test_a_bias_of_the_experts_is_taken(plane):
    for bias in (None, torch.zeros(8), torch.zeros(1, 8), torch.zeros(8, dtype=torch.float64)):
        with pytest.raises(MoEError, match="null context"):
            plane.route_topk(torch.zeros(3, 8), bias=bias)


def test_the_c_entry_point_reports_a_null_context():
    from npu_offload_b200 import _lib
    assert nob.lib().moe_route_topk(None, 1, None, None, None, None, 0, None) == _lib.MOE_EINVAL


# ---------------------------------------------------------------- on the GPU

def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def both(p, logits, bias=None):
    """route_topk against the routing of route(), a context's worth of tokens at a time."""
    idx, w = p.route_topk(logits, bias)
    for a in range(0, logits.shape[0], p.max_tokens):
        r = p.route(logits[a:a + p.max_tokens], bias)
        assert r["status"] == 0
        b = a + p.max_tokens
        assert (idx[a:b].cpu().numpy() == r["idx"]).all() and (w[a:b].cpu().numpy() == r["w"]).all()
    assert idx.shape == w.shape == (logits.shape[0], p.K) and idx.dtype == torch.int32
    assert p.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K", [(8, 2), (33, 1), (128, 8), (160, 6), (256, 16)])
def test_any_number_of_tokens(E, K, scoring):
    """More than the context's max_tokens too, and none."""
    with nob.MoEDataPlane(64, 64, E, K, n_layers=1, max_tokens=64, scoring=scoring) as p:
        g = gen(E + K)
        bias = 0.1 * torch.randn(E, generator=g, device="cuda") if scoring == "sigmoid" else None
        for T in (1, 7, 8, 9, 64, 65, 200):
            both(p, torch.randn(T, E, generator=g, device="cuda") * 3, bias)
        idx, w = p.route_topk(torch.zeros(0, E, device="cuda"))
        assert idx.shape == w.shape == (0, K)
        logits = torch.randn(9000, 2 * E, generator=g, device="cuda")[:, ::2]  # values apart
        idx, w = p.route_topk(logits, bias)
        last = p.route_topk(logits[-5:], bias)
        assert torch.equal(idx[-5:], last[0]) and torch.equal(w[-5:], last[1])
        n = p.launch_count
        p.route_topk(logits, bias)
        assert p.launch_count == n + 1


@pytest.mark.gpu
def test_nan_logits_are_reported():
    from npu_offload_b200._lib import MOE_ENONFINITE, MOE_OK
    with nob.MoEDataPlane(64, 64, 16, 2, n_layers=1, max_tokens=64) as p:
        logits = torch.randn(100, 16, generator=gen(1), device="cuda")
        want = p.route_topk(logits)
        bad = logits.clone()
        bad[70, 3] = float("nan")
        idx, w = p.route_topk(bad)
        assert p.status() == MOE_ENONFINITE and p.status() == MOE_OK
        keep = torch.arange(100, device="cuda") != 70
        assert torch.equal(idx[keep], want[0][keep]) and torch.equal(w[keep], want[1][keep])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 60, 260, 3000])
def test_router_and_experts_in_two_graphs_and_on_two_streams(T):
    """The documented sequence, logits to experts' outputs, run twice at once: neither sees the other's routing."""
    from tests.fp8_util import weight
    H, F, E, K = 256, 128, 32, 4
    with nob.MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=4096) as p:
        g = gen(T)
        gate_up, down = nob.Fp8(*weight(g, E, 2, F, H, spread=H ** -0.5)), nob.Fp8(*weight(g, E, H, F, spread=F ** -0.5))
        args = [(torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16), torch.randn(T, E, generator=g, device="cuda"))
                for _ in range(2)]

        def layer(x, logits):
            idx, w = p.route_topk(logits)
            return idx, w, p.experts_fp8(x, gate_up, down, idx, w)

        want = [layer(*a) for a in args]
        torch.cuda.synchronize()
        assert not torch.equal(want[0][0], want[1][0])
        streams, graphs, outs = [torch.cuda.Stream() for _ in args], [], []
        for s, a in zip(streams, args):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append(layer(*a))
            graphs.append(graph)
        torch.cuda.synchronize()
        for _ in range(20):
            for s, graph, o in zip(streams, graphs, outs):
                with torch.cuda.stream(s):
                    o[2].zero_()
                    graph.replay()
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, v))
        got = [[], []]
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(layer(*args[i]))
        torch.cuda.synchronize()
        for runs, v in zip(got, want):
            assert all(torch.equal(a, b) for r in runs for a, b in zip(r, v))
        assert p.status() == 0
