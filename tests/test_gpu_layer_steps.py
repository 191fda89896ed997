"""The steps around the routed experts run one after the other, as a layer's program calls them: norm, routing in groups, e4m3
experts, the shared expert's products with adapters beside them, the next norm; and the way back of a training step."""
import pytest
import torch

import npu_offload_b200 as nob
from tests.fp8_util import weight
from tests.norm_util import norm64, rounded_sum, scales64
from tests.route_util import choose, weights64

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
H, F, E, K, R, N_AD = 256, 128, 32, 4, 16, 5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Layer:
    def __init__(self, p, g):
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.p = p
        self.norm = (1 + 0.2 * rnd(H)).to(BF), (1 + 0.2 * rnd(H)).to(BF)
        self.router, self.bias = rnd(E, H) * H ** -0.5, 0.05 * rnd(E)
        self.gate_up, self.down = nob.Fp8(*weight(g, E, 2, F, H, spread=H ** -0.5)), nob.Fp8(*weight(g, E, H, F, spread=F ** -0.5))
        self.s_gate_up, self.s_down = nob.Fp8(*weight(g, 2 * F, H, spread=H ** -0.5)), nob.Fp8(*weight(g, H, F, spread=F ** -0.5))
        self.up_a, self.up_b = (rnd(N_AD, R, H) * H ** -0.5).to(BF), (0.1 * rnd(N_AD, 2 * F, R)).to(BF)
        self.dn_a, self.dn_b = (rnd(N_AD, R, F) * F ** -0.5).to(BF), (0.1 * rnd(N_AD, H, R)).to(BF)
        self.scale = 0.5 + torch.rand(N_AD, generator=g, device="cuda")

    def run(self, moe_out, stream, ids):
        """One layer behind the last one's experts: every step's results."""
        p = self.p
        n = p.add_norm(moe_out, self.norm[0], residual=stream, eps=1e-5, fp8=True)
        logits = n.y.float() @ self.router.T
        idx, w = p.route_groups(logits, 8, 3, bias=self.bias, scale=2.5)
        routed = p.experts_fp8(n.y, self.gate_up, self.down, idx, w)
        gu = p.matmul_fp8(n.fp8, self.s_gate_up, out_dtype=F32)
        p.add_lora(gu, n.y, self.up_a, self.up_b, ids, scale=self.scale, out=gu)
        act = (torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]).to(BF)
        shared = p.matmul_fp8(act, self.s_down)
        shared = p.add_lora(shared, act, self.dn_a, self.dn_b, ids, scale=self.scale)
        last = p.add_norm(shared, self.norm[1], residual=n.sum, eps=1e-5)
        return dict(n=n, logits=logits, idx=idx, w=w, routed=routed, gu=gu, act=act, shared=shared, last=last)


def flat(r):
    out = []
    for v in r.values():
        for t in (v if isinstance(v, tuple) else (v,)):
            for u in (t if isinstance(t, tuple) else (t,)):
                if u is not None:
                    out.append(u.view(torch.uint8) if u.dtype == torch.float8_e4m3fn else u)
    return out


def inputs(g, T):
    return (torch.randn(T, H, generator=g, device="cuda"), torch.randn(T, H, generator=g, device="cuda").to(BF),
            torch.randint(-1, N_AD, (T,), generator=g, device="cuda").to(torch.int32))


def product(x, w):
    from tests.fp8_util import expand
    return x @ (w.q.double() * expand(w.scale, w.q.shape, 128)).T


def lora(base, x, a, b, ids, scale):
    out = base.clone()
    for i in range(N_AD):
        t = torch.nonzero(ids == i)[:, 0]
        out[t] += float(scale[i]) * (x[t].double() @ a[i].double().T @ b[i].double().T)
    return out


def near(got, want, part):
    """Off by `part` of the result's size at most."""
    assert float((got.double() - want).norm()) <= part * float(want.norm()), float((got.double() - want).norm() / want.norm())


@pytest.fixture(scope="module")
def plane():
    with nob.MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=16, scoring="sigmoid") as p:
        yield p


@pytest.mark.parametrize("T", [1, 7, 70, 300])
def test_a_layer(plane, T):
    """Each step against 64 bits on what the step before gave: bf16 results to half a step (2^-8 of any value, so of the size),
    with 2^-12 for what was done in fp32 before; a product of values quantised within the call to 2^-4 and 2^-4 more, a
    root-mean-square third of which is left over 256 or 128 terms."""
    g = gen(T)
    layer = Layer(plane, g)
    moe_out, stream, ids = inputs(g, T)
    r = layer.run(moe_out, stream, ids)
    h = rounded_sum(moe_out, stream)
    assert torch.equal(r["n"].sum, h)
    y, rstd = norm64(h, layer.norm[0], 1e-5)
    near(r["n"].y, y, 2.0 ** -8)
    assert torch.equal(r["n"].fp8.scale.double(), scales64(y))
    assert torch.equal(r["idx"].cpu(), choose(r["logits"], 8, 3, K, layer.bias, "sigmoid"))
    near(r["w"], weights64(r["logits"], r["idx"], "sigmoid", True, 2.5), 2.0 ** -16)
    y8 = r["n"].fp8.q.double() * r["n"].fp8.scale.double().repeat_interleave(128, -1)
    base = product(y8, layer.s_gate_up)
    near(r["gu"], lora(base, r["n"].y, layer.up_a, layer.up_b, ids, layer.scale), 2.0 ** -12)
    a8 = plane.quantize_fp8(r["act"])
    base = product(a8.q.double() * a8.scale.double().repeat_interleave(128, -1), layer.s_down)
    near(r["shared"], lora(base, r["act"], layer.dn_a, layer.dn_b, ids, layer.scale), 2.0 ** -7)  # (rounded twice: product, then sum)
    routed = torch.zeros(T, H, device="cuda", dtype=torch.float64)
    for e in torch.unique(r["idx"]).tolist():
        t, k = torch.nonzero(r["idx"] == e, as_tuple=True)
        gu = [product(r["n"].y[t].double(), nob.Fp8(layer.gate_up.q[e, i], layer.gate_up.scale[e, i])) for i in (0, 1)]
        act = torch.nn.functional.silu(gu[0]) * gu[1]
        routed[t] += r["w"][t, k, None].double() * product(act, nob.Fp8(layer.down.q[e], layer.down.scale[e]))
    near(r["routed"], routed, 0.09)
    assert torch.equal(r["last"].sum, rounded_sum(r["shared"], h))
    near(r["last"].y, norm64(r["last"].sum, layer.norm[1], 1e-5)[0], 2.0 ** -8)
    assert plane.status() == 0


@pytest.mark.parametrize("T", [3, 200])
def test_two_layers_at_once_in_graphs_and_on_streams(plane, T):
    g = gen(100 + T)
    layers, data = [Layer(plane, g) for _ in range(2)], [inputs(g, T) for _ in range(2)]
    want = [flat(a.run(*d)) for a, d in zip(layers, data)]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in data], [], []
    for s, a, d in zip(streams, layers, data):
        with torch.cuda.stream(s):
            a.run(*d)  # (torch's own product sets its workspace up outside the capture)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(flat(a.run(*d)))
        graphs.append(graph)
    for _ in range(10):
        for s, graph, o in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                o[0].zero_(), o[-2].zero_()
                graph.replay()
    torch.cuda.synchronize()
    for o, v in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, v))
    assert plane.status() == 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_a_training_step_of_the_router(scoring):
    """The gradient of weights and balance loss, through router and norm, to the residual stream and the norm's weight, against
    autograd in 64 bits with the same choices.  Logits are off by at most (256 + 32) 2^-24 of sum |y| |W| (about 10), so
    the probabilities by 2^-12, and gradients, which are differences of such terms, by 2^-9 of their size."""
    T = 333
    g = gen(7)
    with nob.MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=16, scoring=scoring) as p:
        x, stream = torch.randn(T, H, generator=g, device="cuda"), torch.randn(T, H, generator=g, device="cuda")
        w, router = 1 + 0.2 * torch.randn(H, generator=g, device="cuda"), torch.randn(E, H, generator=g, device="cuda") * H ** -0.5
        dw, ds = torch.randn(T, K, generator=g, device="cuda"), 0.1 * torch.randn(T, H, generator=g, device="cuda")
        n = p.add_norm(x, w, residual=stream, eps=1e-5, out_dtype=F32)
        logits = n.y @ router.T
        idx, top_w = p.route_groups(logits, 8, 3, scale=2.5)
        loss, stats = p.balance_loss(logits, idx)
        dl = p.balance_loss_backward(logits, stats, torch.full((), 3.0, device="cuda"))
        p.route_backward(logits, idx, dw, scale=2.5, out=dl, accumulate=True)
        dx, dweight = p.add_norm_backward(dl @ router, n.sum, w, n.rstd, dsum=ds)
        assert p.status() == 0

        h = n.sum.double().requires_grad_()
        w64 = w.double().requires_grad_()
        l = norm64(h, w64, 1e-5)[0] @ router.double().T
        s = torch.softmax(l, -1) if scoring == "softmax" else torch.sigmoid(l)
        prob = s / s.sum(-1, keepdim=True)
        chosen = s.gather(-1, idx.long())
        weights = 2.5 * chosen / chosen.sum(-1, keepdim=True)
        share = torch.bincount(idx.reshape(-1).long(), minlength=E).double() * E / (K * T)
        total = (weights * dw.double()).sum() + 3 * (share * prob.mean(0)).sum() + (h * ds.double()).sum()
        total.backward()
        near(top_w, weights.detach(), 2.0 ** -12)
        near(dx, h.grad, 2.0 ** -9)
        near(dweight, w64.grad, 2.0 ** -9)
        assert abs(float(loss) - float((share * prob.mean(0)).sum().detach())) < 1e-5
