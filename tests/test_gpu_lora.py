"""Low-rank adapters beside a shared projection, against 64 bits.

Tolerances: the inner sums run over at most K / 128 values one after the other and a few levels more, the outer ones over r;
each step is off by 2^-24 of the sum of sizes |base| + scale sum |x| |a| |b|.  Where results are bf16 the inner sums may be held
in two bf16 parts, 2^-16 together; fp32 ones in three.  The result is rounded once, by half a step of its type."""
import pytest
import torch

import npu_offload_b200 as nob

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def plane():
    with nob.MoEDataPlane(256, 64, 8, 2, n_layers=1, max_tokens=16) as p:
        yield p


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(g, T, K, N, r, n, dtype, ids=None):
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if ids is None:
        ids = torch.randint(-1, n, (T,), generator=g, device="cuda")
    return dict(base=f(T, N).to(dtype), x=f(T, K).to(BF), a=(f(n, r, K) * K ** -0.5).to(BF), b=(f(n, N, r) * r ** -0.5).to(BF), ids=ids.to(torch.int32),
                scale=0.5 + torch.rand(n, generator=g, device="cuda"))


def check(out, base, x, a, b, ids, scale):
    K, r = x.shape[1], a.shape[1]
    want, size = base.double(), base.double().abs()
    for i in torch.unique(ids).tolist():
        if 0 <= i < a.shape[0]:
            t = torch.nonzero(ids == i)[:, 0]
            s = 1.0 if scale is None else float(scale[i])
            want[t] += s * (x[t].double() @ a[i].double().T @ b[i].double().T)
            size[t] += s * (x[t].double().abs() @ a[i].double().abs().T @ b[i].double().abs().T)
    work = (K / 128 + r + 40) * 2.0 ** -24 + (2.0 ** -16 if out.dtype == BF else 0)
    assert out.dtype == base.dtype and out.shape == base.shape
    assert ((out.double() - want).abs() <= torch.finfo(out.dtype).eps / 2 * want.abs() + work * size).all()
    none = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(out[none], base[none])


SHAPES = [(1, 8, 1, 8, 1), (1, 4096, 2560, 16, 8), (2, 64, 3, 8, 2), (3, 72, 40, 24, 3), (7, 1000, 129, 40, 5), (16, 512, 256, 64, 4), (17, 256, 100, 128, 3),
          (33, 136, 77, 16, 40), (64, 1280, 512, 32, 16), (65, 520, 264, 8, 2), (128, 256, 96, 16, 4), (200, 2048, 72, 56, 7), (257, 264, 1283, 16, 1),
          (300, 640, 320, 64, 300), (513, 128, 2056, 120, 3), (1000, 1032, 200, 16, 33), (1500, 4096, 64, 8, 3), (130, 8192, 33, 128, 2)]


@pytest.mark.parametrize("T,K,N,r,n", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_adapters(plane, T, K, N, r, n, dtype):
    g = gen(T + K + N)
    m = make(g, T, K, N, r, n, dtype)
    if T == 1:
        m["ids"].zero_()
    check(plane.add_lora(**m), **m)
    m["scale"] = None
    check(plane.add_lora(**m), **m)
    assert plane.status() == 0


@pytest.mark.parametrize("T", [5, 70, 700])
@pytest.mark.parametrize("kind", ["runs", "one", "none", "last", "own"])
def test_how_tokens_share_adapters(plane, T, kind):
    g = gen(T)
    n = 2000 if kind == "own" else 6
    ids = {"runs": torch.arange(T, device="cuda") * 6 // T, "one": torch.full((T,), 3, device="cuda"), "none": torch.full((T,), -1, device="cuda"),
           "last": torch.where(torch.arange(T, device="cuda") == T - 1, 5, -1), "own": torch.randperm(n, generator=g, device="cuda")[:T]}[kind]
    m = make(g, T, 160, 136, 16, n, BF, ids)
    out = plane.add_lora(**m)
    check(out, **m)
    assert torch.equal(plane.add_lora(**m), out)  # no sum depends on timing
    base = m["base"].clone()
    assert plane.add_lora(**{**m, "base": base}, out=base).data_ptr() == base.data_ptr() and torch.equal(base, out)


@pytest.mark.parametrize("T", [6, 400])
def test_ids_out_of_range(plane, T):
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    m = make(gen(1), T, 64, 48, 8, 4, F32)
    m["ids"][1], m["ids"][T - 1], m["ids"][0] = 4, 2 ** 31 - 1, -2 ** 31
    out = plane.add_lora(**m)
    assert plane.status() == MOE_EINVAL and plane.status() == MOE_OK
    check(out, **m)


@pytest.mark.parametrize("T", [4, 300])
def test_special_values_stay_in_their_token(plane, T):
    m = make(gen(2), T, 128, 64, 16, 3, F32)
    m["ids"][0], m["ids"][1], m["ids"][2] = 1, -1, 1
    want = plane.add_lora(**m)
    x = m["x"].clone()
    x[0, 5] = float("inf")
    x[1] = float("nan")  # a token without an adapter: nothing of it is used
    a = m["a"].clone()
    a[2, 0, 0] = float("nan")
    m["ids"][m["ids"] == 2] = 0
    want = plane.add_lora(**m)
    got = plane.add_lora(**{**m, "x": x, "a": a})
    assert not got[0].isfinite().all() and torch.equal(got[1:], want[1:])
    # an infinity in x: low is one, of a sign or the other, or NaN, and so is the sum of its products with B
    low = (x[0].double()[None] @ m["a"][1].double().T) * float(m["scale"][1])
    exact = m["base"][0].double() + (low @ m["b"][1].double().T)[0]
    assert torch.equal(got[0].isnan(), exact.isnan()) and torch.equal(got[0][~exact.isnan()].double(), exact[~exact.isnan()])


def test_strides_no_tokens_and_wide_rows(plane):
    g = gen(3)
    m = make(g, 20, 256, 72, 16, 4, BF)
    wide = torch.randn(20, 512, generator=g, device="cuda").to(BF)
    m["x"] = wide[:, ::2]
    check(plane.add_lora(**m), **m)
    m["base"] = torch.randn(72, 20, generator=g, device="cuda").T
    check(plane.add_lora(**m), **m)
    empty = make(g, 0, 256, 72, 16, 4, BF, torch.zeros(0, device="cuda"))
    assert plane.add_lora(**empty).shape == (0, 72)
    before = plane.launch_count
    none = dict(base=torch.zeros(5, 0, device="cuda"), x=torch.zeros(5, 64, device="cuda", dtype=BF), a=torch.zeros(1, 8, 64, device="cuda", dtype=BF),
                b=torch.zeros(1, 0, 8, device="cuda", dtype=BF), ids=torch.zeros(5, device="cuda", dtype=torch.int32))
    assert plane.add_lora(**none).shape == (5, 0) and plane.launch_count == before


@pytest.mark.parametrize("T", [9, 600])
def test_another_stream_and_captured_graphs(plane, T):
    g = gen(T)
    data = [make(g, T, 320, 264, 32, 5, BF) for _ in range(2)]
    want = [plane.add_lora(**m) for m in data]
    torch.cuda.synchronize()
    other = plane.add_lora(**data[0], stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    assert torch.equal(other, want[0])
    streams, graphs, outs = [torch.cuda.Stream() for _ in data], [], []
    for s, m in zip(streams, data):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(plane.add_lora(**m))
        graphs.append(graph)
    for _ in range(20):
        for s, graph, o in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                o.zero_()
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # a replay goes by what its inputs hold by then
    data[0]["ids"].copy_(torch.randint(-1, 5, (T,), generator=g, device="cuda"))
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], **data[0])


def test_the_library_refuses(plane):
    from npu_offload_b200 import _lib
    L = nob.lib()
    m = make(gen(4), 4, 64, 32, 8, 2, BF)
    out, ws, p = torch.zeros(4, 32, device="cuda", dtype=BF), torch.zeros(1 << 20, device="cuda"), lambda t: t.data_ptr()
    before = plane.launch_count

    def call(T=4, K=64, N=32, r=8, n=2, base=p(m["base"]), x=p(m["x"]), o=p(out), dt=0, flags=0):
        return L.moe_add_lora(plane.handle, T, K, N, r, n, base, x, p(m["a"]), p(m["b"]), p(m["ids"]), None, o, dt, p(ws), 1 << 22, flags, None)

    for kw, needle in ((dict(T=-1), "T="), (dict(T=(1 << 20) + 1), "T="), (dict(K=0), "K="), (dict(K=60), "K="), (dict(N=-1), "N="), (dict(r=0), "r="),
                       (dict(r=12), "r="), (dict(r=136), "r="), (dict(n=0), "n="), (dict(n=4097), "n="), (dict(dt=2), "out_dtype"), (dict(x=None), "null"),
                       (dict(o=None), "null"), (dict(x=p(m["x"]) + 2), "aligned"), (dict(o=p(m["x"])), "overlaps"), (dict(o=p(m["base"]) + 16), "overlaps"),
                       (dict(flags=2), "flag")):
        assert call(**kw) == _lib.MOE_EINVAL and needle in _lib.last_error(), kw
    assert plane.launch_count == before
    for bad in ((1 << 21, 8, 1), (1, 8, 0), (1, 0, 1), (-1, 8, 1)):
        assert L.moe_add_lora_workspace(plane.handle, *bad) == -1


@pytest.mark.parametrize("r,tokens", [(32, 128), (64, 64), (128, 32)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("more", [0, 1])
def test_on_both_sides_of_few_tokens(plane, r, tokens, dtype, more):
    """One kernel on one side, three on the other; columns that end inside a warp's and a block's."""
    m = make(gen(r + more), tokens + more, 328, 300, r, 3, dtype)
    check(plane.add_lora(**m), **m)


@pytest.mark.parametrize("r", [16, 64, 128])
@pytest.mark.parametrize("last", [1, 16, 17, 32, 33, 48, 49, 64])
def test_tiles_that_end_anywhere(plane, r, last):
    """Tokens of one adapter beyond whole tiles of 64: rows behind a tile's last are no one's."""
    T = 192 + last
    m = make(gen(r + last), T, 136, 264, r, 2, BF)
    m["ids"] = torch.zeros(T, dtype=torch.int32, device="cuda")
    check(plane.add_lora(**m), **m)
    m["ids"].fill_(1)
    m["ids"][5] = -1
    check(plane.add_lora(**m), **m)
    assert plane.status() == 0


@pytest.mark.parametrize("T,K,N,r,n", [(4096, 264, 136, 64, 32), (2500, 4096, 40, 128, 64), (5000, 136, 72, 104, 3)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_more_tiles_than_run_at_once(plane, T, K, N, r, n, dtype):
    """Of higher ranks, a tile then has fewer CTAs and a CTA a larger share of the inner dimension."""
    m = make(gen(T + r), T, K, N, r, n, dtype)
    check(plane.add_lora(**m), **m)
    assert plane.status() == 0
