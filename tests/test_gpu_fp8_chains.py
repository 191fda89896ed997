"""Kernels that start ahead of the end of the ones before them: calls whose outputs are the next call's operands, written
into the same buffers time and again with nothing between them that would hold the next one back."""
import pytest
import torch

from tests.fp8_util import EPS, weight

pytestmark = pytest.mark.gpu

# (tokens, experts, choices): up to 32 pairs, up to 1024, more; groups of 16, 32 and 128 rows
SIZES = [(1, 16, 4), (6, 16, 4), (60, 16, 4), (200, 16, 4), (500, 16, 4), (40, 64, 8), (300, 128, 8), (700, 8, 2)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


class Chain:
    """Features -> product -> tokens; features -> product -> logits -> routing; weights -> quantiser; all -> experts."""

    def __init__(self, T, E, K, seed=0):
        from npu_offload_b200 import Fp8, MoEDataPlane
        self.H, self.F, self.T, self.E, self.K = 256, 192, T, E, K
        self.p = MoEDataPlane(self.H, self.F, E, K, n_layers=1, max_tokens=16)
        g = gen(seed + T)
        self.features = [self.p.quantize_fp8(randn(g, T, 512)) for _ in range(3)]
        self.to_x, self.to_logits = (Fp8(*weight(g, n, 512, spread=512 ** -0.5)) for n in (self.H, E))
        self.gate_up = [(randn(g, E, 2, self.F, self.H) * self.H ** -0.5).to(torch.bfloat16) for _ in range(3)]
        self.down = [(randn(g, E, self.H, self.F) * self.F ** -0.5).to(torch.bfloat16) for _ in range(3)]
        self.x = torch.zeros(T, self.H, dtype=torch.bfloat16, device="cuda")
        self.logits = torch.zeros(T, E, device="cuda")
        self.out = torch.zeros(T, self.H, device="cuda")

    def step(self, i, wait=lambda: None):
        """One pass on the i-th inputs; wait() stands between its calls."""
        p = self.p
        p.matmul_fp8(self.features[i], self.to_logits, out=self.logits)
        wait()
        gate_up = p.quantize_fp8(self.gate_up[i], block_rows=128)
        wait()
        idx, w = p.route_topk(self.logits)
        wait()
        p.matmul_fp8(self.features[i], self.to_x, out=self.x)
        wait()
        down = p.quantize_fp8(self.down[i], block_rows=128)
        wait()
        y = p.experts_fp8(self.x, gate_up, down, idx, w)
        wait()
        p.experts_fp8(self.x, gate_up, down, idx, w, out=self.out, accumulate=True)
        wait()
        return y


@pytest.mark.parametrize("T,E,K", SIZES)
def test_operands_written_by_the_call_before(T, E, K):
    c = Chain(T, E, K)
    try:
        want, sums = [], []
        for i in range(3):
            c.out.zero_()
            want.append(c.step(i, torch.cuda.synchronize))
            sums.append(c.out.clone())
        assert not torch.equal(want[0], want[1])
        # the sum starts at what out held, 0
        assert all(torch.equal(s, y) for s, y in zip(sums, want))
        got = []
        for n in range(30):  # temporaries of one pass are the buffers of the next
            got.append((n % 3, c.step(n % 3)))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i, y in got)
        assert c.p.status() == 0
    finally:
        c.p.close()


@pytest.mark.parametrize("T,E,K", SIZES)
def test_the_same_in_a_captured_graph(T, E, K):
    c = Chain(T, E, K, seed=1)
    try:
        want = [c.step(i, torch.cuda.synchronize) for i in range(3)]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = [c.step(n % 3) for n in range(6)]
        for _ in range(5):
            for y in got:
                y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(y, want[n % 3]) for n, y in enumerate(got))
        assert c.p.status() == 0
    finally:
        c.p.close()


@pytest.mark.parametrize("T,E,K", [(1, 16, 4), (60, 16, 4), (500, 16, 4)])
def test_sums_over_calls_that_follow_at_once(T, E, K):
    """out += of several calls one behind the other: each reads the sum that the one before it left."""
    c = Chain(T, E, K, seed=2)
    try:
        ys = [c.step(i, torch.cuda.synchronize) for i in range(1)]
        gate_up, down = (c.p.quantize_fp8(m[0], block_rows=128) for m in (c.gate_up, c.down))
        idx, w = c.p.route_topk(c.logits)
        c.out.zero_()
        n = 12
        for _ in range(n):
            c.p.experts_fp8(c.x, gate_up, down, idx, w, out=c.out, accumulate=True)
        torch.cuda.synchronize()
        # choices are added to the sum one by one, K of them a call: K n roundings of numbers up to the sum of magnitudes
        mag = torch.zeros_like(c.out, dtype=torch.float64)
        for k in range(K):
            one = torch.full_like(idx, -1)
            one[:, k] = idx[:, k]
            mag += c.p.experts_fp8(c.x, gate_up, down, one, w).double().abs()
        assert bool(((c.out.double() - n * ys[0].double()).abs() <= (K * n + K * n) * EPS * n * mag).all())
        assert c.p.status() == 0
    finally:
        c.p.close()
