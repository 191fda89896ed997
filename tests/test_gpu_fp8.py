"""e4m3 quantiser, scaled product and routed experts on the GPU against their 64-bit definitions."""
import pytest
import torch

from tests.fp8_util import EPS, F8, ceil128, experts64, expand, matmul64, matmul_bound, quantize64, weight

pytestmark = pytest.mark.gpu
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


@pytest.fixture(scope="module")
def planes():
    from npu_offload_b200 import MoEDataPlane
    cache = {}

    def get(H=256, F=64, E=8, K=2, **kw):
        key = (H, F, E, K, tuple(sorted(kw.items())))
        if key not in cache:
            cache[key] = MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=16, **kw)
        return cache[key]
    yield get
    for p in cache.values():
        p.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(b, nan=1e9))


# ---------------------------------------------------------------- quantiser

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,block_rows", [
    ((1, 16), 1), ((1, 4096), 1), ((3, 144), 1), ((1000, 272), 1), ((4099, 1280), 1), ((2, 3, 5, 112), 1),
    ((1, 16), 128), ((128, 128), 128), ((129, 144), 128), ((3, 2, 64, 256), 128), ((300, 2000), 128)])
def test_quantize_is_the_definition(planes, shape, block_rows, dtype):
    g = gen(sum(shape) + block_rows)
    x = (randn(g, *shape) * torch.exp(4 * randn(g, *shape[:-1], 1))).to(dtype)
    got = planes().quantize_fp8(x, block_rows=block_rows)
    q, s = quantize64(x, block_rows)
    assert torch.equal(got.scale.double(), s)
    assert same(got.q.double(), q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_of_extreme_values(planes, block_rows, dtype):
    """Zeros, infinities, NaN, the smallest and largest numbers, maxima at a change of scale, ties."""
    rows = torch.zeros(10, 256, device="cuda")
    g = gen(3)
    rows[1] = randn(g, 256)
    rows[1, 5], rows[1, 200] = float("inf"), float("-inf")
    rows[2] = randn(g, 256)
    rows[2, 0] = float("nan")
    rows[3] = float("inf")
    rows[4] = randn(g, 256).sign() * 2.0 ** -133
    rows[5] = randn(g, 256) * 1e38
    rows[6] = torch.linspace(-448, 448, 256, device="cuda")
    rows[7] = torch.linspace(-450, 450, 256, device="cuda")
    rows[8] = torch.arange(256, device="cuda") * 2.0 ** -10  # halves of the smallest steps
    rows[8, 128] = rows[8, 0] = 448
    rows[9, 3] = -0.0
    x = rows.to(dtype)
    got = planes().quantize_fp8(x, block_rows=block_rows)
    q, s = quantize64(x, block_rows)
    assert torch.equal(got.scale.double(), s)
    assert same(got.q.double(), q)


def test_quantize_of_views_and_nothing(planes):
    p = planes()
    x = randn(gen(1), 65, 80)
    for v in (x[:, 16:64], x[1:, :].T[:, :64], x.flatten()[1:1 + 64 * 16].view(64, 16)):  # strides, an odd address
        assert same(p.quantize_fp8(v).q.double(), quantize64(v, 1)[0])
    for shape in ((0, 32), (4, 0), (0, 3, 32)):
        r = p.quantize_fp8(torch.zeros(shape, device="cuda"))
        assert r.q.shape == shape and r.scale.numel() == 0
    from npu_offload_b200._lib import MoEError
    with pytest.raises(MoEError, match="multiple of 16"):
        p.quantize_fp8(torch.zeros(4, 24, device="cuda"))
    with pytest.raises(ValueError, match="tensor on"):
        p.quantize_fp8(torch.zeros(4, 32))


# ---------------------------------------------------------------- product

def product(p, M, N, K, out_dtype, seed, general=True):
    g = gen(seed)
    x = p.quantize_fp8(randn(g, M, K) * torch.exp(2 * randn(g, M, 1)))
    w = weight(g, N, K, general=general)
    from npu_offload_b200 import Fp8
    out = p.matmul_fp8(x, Fp8(*w), out_dtype=out_dtype)
    want, mag = matmul64(*x, *w)
    bound = matmul_bound(mag, K)
    if out_dtype == torch.bfloat16:
        bound = bound + BF16_HALF * (want.abs() + bound)
    off = (out.double() - want).abs() - bound
    assert out.dtype == out_dtype and out.shape == (M, N)
    assert bool((off <= 0).all()), (M, N, K, float(off.max()), float(want.abs().max()))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 128, 128), (1, 129, 144), (2, 33, 4096), (5, 2560, 1024), (16, 16, 16), (17, 300, 272),
    (31, 127, 2048), (64, 384, 640), (65, 255, 112), (100, 1000, 1008), (128, 128, 256), (129, 257, 384),
    (200, 1280, 528), (300, 511, 1280), (777, 513, 208), (1, 4096, 16384), (40, 200, 16384), (200, 200, 16384)])
def test_matmul_is_the_definition(planes, M, N, K, out_dtype):
    product(planes(), M, N, K, out_dtype, M + N + K)


@pytest.mark.parametrize("M", list(range(1, 70, 3)) + [96, 97, 127, 160, 192, 255, 256, 257])
def test_matmul_over_the_number_of_rows(planes, M):
    product(planes(), M, 400, 400, torch.float32, M)


def test_matmul_of_large_operands(planes):
    """Against 64 bits at sizes with many tiles, and the last rows and columns of each."""
    product(planes(), 2049, 1921, 1152, torch.float32, 5)
    product(planes(), 1023, 4097, 512, torch.bfloat16, 6)


def test_matmul_of_extreme_scales_and_nan(planes):
    """Scales of either end, rows of NaN and infinity: other rows and columns do not see them."""
    from npu_offload_b200 import Fp8
    p, g = planes(), gen(9)
    for M in (7, 150):
        x = p.quantize_fp8(randn(g, M, 384))
        x.scale[0] = 2.0 ** 80
        x.scale[1] = 2.0 ** -80
        x.scale[2] = float("inf")
        w, ws = weight(g, 200, 384)
        xn = x.q.clone()
        xn.view(torch.uint8)[3, 200] = 0x7f  # NaN
        wn = w.clone()
        wn.view(torch.uint8)[140, 5] = 0xff
        out = p.matmul_fp8(Fp8(xn, x.scale), Fp8(wn, ws), out_dtype=torch.float32)
        want, mag = matmul64(xn, x.scale, wn, ws)
        assert out[3].isnan().all() and out[:, 140].isnan().all()
        ok = torch.ones_like(want, dtype=torch.bool)
        ok[2:4], ok[:, 140] = False, False
        bound = matmul_bound(mag, 384)
        assert bool(((out.double() - want).abs() <= bound)[ok].all())
        assert not out[2].isfinite().any()


def test_matmul_takes_unquantised_rows_and_an_out(planes):
    from npu_offload_b200 import Fp8
    p, g = planes(), gen(4)
    x = randn(g, 9, 256).to(torch.bfloat16)
    w = Fp8(*weight(g, 130, 256))
    a = p.matmul_fp8(p.quantize_fp8(x), w)
    assert torch.equal(a, p.matmul_fp8(x, w))
    out = torch.full((9, 130), 7.0, device="cuda")
    assert p.matmul_fp8(x, w, out=out) is out and torch.equal(out.to(torch.bfloat16), a)
    # rows behind the output are left as they were
    big = torch.full((12, 130 * 8), 7.0, device="cuda")
    view = big.view(-1)[:9 * 130].view(9, 130)
    p.matmul_fp8(x, w, out=view)
    assert torch.equal(view, out) and bool((big.view(-1)[9 * 130:] == 7).all())


def test_matmul_of_nothing_and_refusals(planes):
    from npu_offload_b200 import Fp8
    from npu_offload_b200._lib import MoEError
    p = planes()
    w = Fp8(*weight(gen(1), 32, 64))
    assert p.matmul_fp8(p.quantize_fp8(torch.zeros(0, 64, device="cuda")), w).shape == (0, 32)
    e = Fp8(torch.zeros(0, 64, device="cuda").to(F8), torch.zeros(0, 1, device="cuda"))
    assert p.matmul_fp8(torch.zeros(3, 64, device="cuda"), e).shape == (3, 0)
    for K in (24, 16400):
        x = Fp8(torch.zeros(1, K, device="cuda").to(F8), torch.ones(1, ceil128(K), device="cuda"))
        with pytest.raises(MoEError, match="multiple of 16 in"):
            p.matmul_fp8(x, Fp8(torch.zeros(1, K, device="cuda").to(F8), torch.ones(1, ceil128(K), device="cuda")))


def test_matmul_is_the_same_every_time_and_in_a_graph(planes):
    from npu_offload_b200 import Fp8
    p, g = planes(), gen(8)
    for M in (1, 20, 300):
        x, w = p.quantize_fp8(randn(g, M, 2048)), Fp8(*weight(g, 640, 2048))
        first = p.matmul_fp8(x, w, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(first, p.matmul_fp8(x, w, out_dtype=torch.float32))
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = p.matmul_fp8(x, w, out_dtype=torch.float32)
        torch.cuda.synchronize()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(first, out)
    assert p.status() == 0


# ---------------------------------------------------------------- experts

def expert_case(seed, T, H, F, E, K, general=True, spread=None):
    g = gen(seed)
    x = (randn(g, T, H)).to(torch.bfloat16)
    gu = weight(g, E, 2, F, H, general=general, spread=spread or H ** -0.5)
    d = weight(g, E, H, F, general=general, spread=spread or F ** -0.5)
    p, idx = torch.softmax(randn(g, T, E) - torch.log(torch.arange(E, device="cuda") + 1.0), -1).topk(K, -1)
    return x, gu, d, idx.int().contiguous(), (p / p.sum(-1, keepdim=True)).contiguous()


def check_experts(p, x, gu, d, idx, w, out_dtype=torch.float32):
    from npu_offload_b200 import Fp8
    out = p.experts_fp8(x, Fp8(*gu), Fp8(*d), idx, w, out_dtype=out_dtype)
    assert p.status() == 0
    want, bound = experts64(x, *gu, *d, idx, w)
    if out_dtype == torch.bfloat16:
        bound = bound + BF16_HALF * (want.abs() + bound)
    off = (out.double() - want).abs() - bound
    assert out.dtype == out_dtype and bool((off <= 0).all()), (float(off.max()), float(want.abs().max()))
    # the bound is no licence: few values may lie near a border
    assert float((out.double() - want).norm()) <= 0.01 * float(want.norm()) + 1e-30
    return out


@pytest.mark.parametrize("T,H,F,E,K", [
    (1, 256, 64, 8, 2), (1, 4096, 1280, 16, 8), (2, 64, 64, 1, 1), (3, 320, 192, 60, 6), (7, 1024, 128, 4, 4),
    (16, 512, 256, 128, 8), (17, 192, 320, 8, 1), (40, 256, 128, 2, 2), (70, 128, 64, 1, 1), (130, 384, 256, 3, 2),
    (300, 256, 192, 8, 2), (600, 128, 128, 2, 1)])
def test_experts_are_the_definition(planes, T, H, F, E, K):
    check_experts(planes(H, F, E, K), *expert_case(T + H + F + E, T, H, F, E, K))


@pytest.mark.parametrize("T", [1, 5, 33, 64, 90])
def test_experts_into_bf16(planes, T):
    check_experts(planes(256, 128, 8, 4), *expert_case(T, T, 256, 128, 8, 4), out_dtype=torch.bfloat16)


@pytest.mark.parametrize("T", [1, 9, 150])
def test_experts_with_choices_left_out(planes, T):
    """Negative choices, tokens with none at all (their output is zero), an expert chosen twice by a token."""
    p = planes(256, 128, 8, 4)
    x, gu, d, idx, w = expert_case(50 + T, T, 256, 128, 8, 4)
    idx[0] = torch.tensor([3, -1, 3, -7], device="cuda", dtype=torch.int32)
    w[0, 1] = float("nan")  # the weight of no expert is not looked at
    if T > 1:
        idx[T // 2] = -1
        idx[T - 1, 1:] = -1
    out = check_experts(p, x, gu, d, idx, w)
    if T > 1:
        assert bool((out[T // 2] == 0).all())
    idx[:] = -1
    assert bool((check_experts(p, x, gu, d, idx, w) == 0).all())


def test_experts_accumulate_and_leave_the_rest(planes):
    from npu_offload_b200 import Fp8
    p = planes(256, 128, 8, 4)
    for T in (3, 140):
        x, gu, d, idx, w = expert_case(T, T, 256, 128, 8, 4)
        gu, d = Fp8(*gu), Fp8(*d)
        plain = p.experts_fp8(x, gu, d, idx, w)
        big = torch.full((T + 2, 256), 3.0, device="cuda")
        p.experts_fp8(x, gu, d, idx, w, out=big[:T], accumulate=True)
        assert bool(((big[:T] - plain - 3).abs() <= 4 * EPS * (plain.abs() + 6)).all())
        assert bool((big[T:] == 3).all())
        from npu_offload_b200._lib import MoEError
        with pytest.raises(MoEError, match="fp32"):
            p.experts_fp8(x, gu, d, idx, w, out=big[:T].to(torch.bfloat16), accumulate=True)


def test_experts_report_an_index_out_of_range(planes):
    from npu_offload_b200 import Fp8
    from npu_offload_b200._lib import MOE_EINVAL, MOE_OK
    p = planes(256, 128, 8, 4)
    for T in (2, 100):
        x, gu, d, idx, w = expert_case(T, T, 256, 128, 8, 4)
        bad = idx.clone()
        bad[1, 2] = 8
        bad[0, 0] = 2 ** 31 - 1
        out = p.experts_fp8(x, Fp8(*gu), Fp8(*d), bad, w)
        assert p.status() == MOE_EINVAL and p.status() == MOE_OK
        none = torch.where((bad < 0) | (bad >= 8), -1, bad).int()
        assert torch.equal(out, p.experts_fp8(x, Fp8(*gu), Fp8(*d), none, w))


def test_experts_of_nan_and_infinity_stay_in_their_rows(planes):
    from npu_offload_b200 import Fp8
    p = planes(256, 128, 8, 4)
    for T in (6, 80):
        x, gu, d, idx, w = expert_case(T, T, 256, 128, 8, 4)
        clean = p.experts_fp8(x, Fp8(*gu), Fp8(*d), idx, w)
        x[2, 3], x[4, 100] = float("nan"), float("inf")
        out = p.experts_fp8(x, Fp8(*gu), Fp8(*d), idx, w)
        assert out[2].isnan().all() and out[4].isnan().all()
        rest = [t for t in range(T) if t not in (2, 4)]
        assert torch.equal(out[rest], clean[rest])
    assert p.status() == 0


def test_experts_of_nothing(planes):
    from npu_offload_b200 import Fp8
    p = planes(256, 128, 8, 4)
    x, gu, d, idx, w = expert_case(1, 1, 256, 128, 8, 4)
    assert p.experts_fp8(x[:0], Fp8(*gu), Fp8(*d), idx[:0], w[:0]).shape == (0, 256)


def test_two_graphs_and_two_streams_at_once(planes):
    """Calls in two captured graphs, replayed at once on two streams, do not share working memory."""
    from npu_offload_b200 import Fp8
    p = planes(512, 256, 16, 4)
    for T in (4, 260):
        cases = [expert_case(70 + i + T, T, 512, 256, 16, 4) for i in range(2)]
        args = [(x, Fp8(*gu), Fp8(*d), idx, w) for x, gu, d, idx, w in cases]
        want = [p.experts_fp8(*a) for a in args]
        streams, graphs, outs = [torch.cuda.Stream() for _ in args], [], []
        torch.cuda.synchronize()
        for s, a in zip(streams, args):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append(p.experts_fp8(*a))
            graphs.append(graph)
        torch.cuda.synchronize()
        for _ in range(10):
            for s, graph, o in zip(streams, graphs, outs):
                with torch.cuda.stream(s):
                    o.zero_()
                    graph.replay()
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert torch.equal(o, v)
        got = []
        for s, a in zip(streams, args):
            s.wait_stream(torch.cuda.current_stream())
            got.append([p.experts_fp8(*a, stream=s) for _ in range(5)])
        torch.cuda.synchronize()
        for rs, v in zip(got, want):
            assert all(torch.equal(r, v) for r in rs)
    assert p.status() == 0


def test_a_layer_as_it_is_used(planes):
    """Router, experts, shared expert's product and residual in one run, on quantised weights."""
    from npu_offload_b200 import Fp8
    H, F, E, K, T = 512, 256, 16, 4, 11
    p, g = planes(H, F, E, K), gen(77)
    x = randn(g, T, H).to(torch.bfloat16)
    gate_up = p.quantize_fp8((randn(g, E, 2, F, H) * H ** -0.5).to(torch.bfloat16), block_rows=128)
    down = p.quantize_fp8((randn(g, E, H, F) * F ** -0.5).to(torch.bfloat16), block_rows=128)
    shared = p.quantize_fp8(randn(g, H, H) * H ** -0.5, block_rows=128)
    logits = randn(g, T, E)
    idx, w = p.route_topk(logits)
    r = p.route(logits)
    assert (idx.cpu().numpy() == r["idx"]).all() and (w.cpu().numpy() == r["w"]).all()
    out = p.experts_fp8(x, gate_up, down, idx, w)
    want, bound = experts64(x, *gate_up, *down, idx, w)
    assert bool(((out.double() - want).abs() <= bound).all())
    p.matmul_fp8(x, shared, out_dtype=torch.float32)
    nxt = p.combine_residual(p.matmul_fp8(x, shared), out)
    xq = p.quantize_fp8(x)
    y, mag = matmul64(*xq, *shared)
    e = matmul_bound(mag, H) + BF16_HALF * y.abs() * 1.01
    total = y + want
    lim = bound + e + 2 * EPS * (y.abs() + want.abs())
    assert bool(((nxt.double() - total).abs() <= lim + BF16_HALF * (total.abs() + lim)).all())
    loss, stats = p.balance_loss(logits, idx)
    assert int(stats.counts.sum()) == T * K and float(loss) > 0
    assert p.status() == 0


def test_calls_leave_the_current_device_and_do_not_wait(planes):
    p = planes()
    before = torch.cuda.current_device()
    n = p.launch_count
    p.quantize_fp8(torch.ones(2, 32, device="cuda"))
    assert torch.cuda.current_device() == before and p.launch_count == n + 1


# ---------------------------------------------------------------- sizes at which another kernel takes over

@pytest.mark.parametrize("M,K", [(8, 512), (8, 640), (9, 1280), (9, 1296), (16, 1408), (17, 2048), (17, 2064), (32, 2176), (33, 4096),
                                 (33, 4112), (64, 4096), (64, 4224), (65, 4224)])
def test_matmul_either_side_of_a_change_of_kernel(planes, M, K):
    product(planes(), M, 385, K, torch.float32, M + K)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(2049, 1921, 16), (2049, 1922, 144), (2048, 2560, 272), (1025, 6148, 400), (1, 65537, 48), (5000, 24, 160)])
def test_matmul_of_many_tiles_and_few_blocks(planes, M, N, K, out_dtype):
    """Rows of every alignment, tiles of either width, one to four blocks a tile and more tiles than SMs."""
    product(planes(), M, N, K, out_dtype, N + K)


@pytest.mark.parametrize("M", [3, 12, 40, 100])
def test_nan_and_infinity_stay_what_they_are_in_bf16(planes, M):
    from npu_offload_b200 import Fp8
    p, g = planes(), gen(M)
    x = p.quantize_fp8(randn(g, M, 256))
    w = weight(g, 136, 256)
    bad = x.q.clone()
    bad.view(torch.uint8)[1] = 0x7f
    scale = x.scale.clone()
    scale[2] = 3e38  # products beyond the largest bf16
    out = p.matmul_fp8(Fp8(bad, scale), Fp8(*w))
    assert out[1].isnan().all()
    # a block's sum beyond the largest number: the result is not finite; of one sign, it is that infinity (of both,
    # the infinity of the one added first or NaN, as the second is added by a fused operation or a plain one)
    blocks = [matmul64(bad[:, k:k + 128], scale[:, k // 128:k // 128 + 1], w[0][:, k:k + 128], w[1][:, k // 128:k // 128 + 1])[0][2]
              for k in (0, 128)]
    far = [b.abs() >= (2 - 2.0 ** -24) * 2.0 ** 127 for b in blocks]  # what rounds beyond the largest number
    assert far[0].any() and far[1].any()
    sums = sum(torch.where(f, b.sign() * float("inf"), 0.0) for f, b in zip(far, blocks))
    over = far[0] | far[1]
    assert not out[2][over].isfinite().any()
    assert torch.equal(out[2][sums.isinf()].double(), sums[sums.isinf()])
    assert torch.equal(out[0], p.matmul_fp8(x, Fp8(*w))[0])


@pytest.mark.parametrize("T,H,F,E,K", [(520, 128, 64, 8, 2), (300, 128, 128, 128, 8), (1100, 64, 64, 60, 1), (129, 64, 64, 3, 8 // 4),
                                       (2049, 64, 64, 1, 1), (1024, 64, 64, 256, 1), (1025, 64, 64, 256, 1)])
def test_experts_of_many_pairs(planes, T, H, F, E, K):
    """More pairs than one CTA groups, experts with many groups of rows and with none."""
    check_experts(planes(H, F, E, K), *expert_case(T + E, T, H, F, E, K))


def test_experts_of_many_pairs_with_choices_left_out(planes):
    from npu_offload_b200._lib import MOE_EINVAL
    from npu_offload_b200 import Fp8
    p = planes(64, 64, 8, 4)
    x, gu, d, idx, w = expert_case(3, 500, 64, 64, 8, 4)
    g = gen(12)
    idx[torch.rand(500, 4, generator=g, device="cuda") < 0.4] = -1
    idx[100:140] = -1
    out = check_experts(p, x, gu, d, idx, w)
    assert bool((out[100:140] == 0).all())
    bad = idx.clone()
    bad[7, 1] = 8
    assert torch.equal(p.experts_fp8(x, Fp8(*gu), Fp8(*d), bad, w)[8:], out[8:]) and p.status() == MOE_EINVAL
    idx[:] = -1
    assert bool((check_experts(p, x, gu, d, idx, w) == 0).all())


# ---------------------------------------------------------------- order, waits

def test_results_follow_the_order_of_the_stream(planes):
    """Kernels are launched ahead of the end of the ones before them: inputs written just before a call, and
    overwritten just after it, are the call's own; so are weights, results and working memory taken over."""
    from npu_offload_b200 import Fp8
    p, g = planes(512, 256, 16, 4), gen(21)
    for T in (2, 30, 300):
        cases = [expert_case(900 + i, T, 512, 256, 16, 4) for i in range(3)]
        want = [p.experts_fp8(x, Fp8(*gu), Fp8(*d), idx, w) for x, gu, d, idx, w in cases]
        torch.cuda.synchronize()
        buf = [[t.clone() if isinstance(t, torch.Tensor) else [u.clone() for u in t] for t in c] for c in cases[:1]][0]
        got = []
        for _ in range(4):
            for c in cases:
                for dst, src in zip(buf, c):
                    for a, b in zip(*(([dst], [src]) if isinstance(dst, torch.Tensor) else (dst, src))):
                        a.view(torch.uint8).copy_(b.view(torch.uint8)) if a.dtype == F8 else a.copy_(b)
                got.append(p.experts_fp8(buf[0], Fp8(*buf[1]), Fp8(*buf[2]), buf[3], buf[4]))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(got))
    xs = [randn(g, 40, 2048) for _ in range(3)]
    w = Fp8(*weight(g, 300, 2048))
    want = [p.matmul_fp8(x, w) for x in xs]
    buf, got = torch.empty_like(xs[0]), []
    for i in range(12):
        buf.copy_(xs[i % 3])
        got.append(p.matmul_fp8(buf, w))
    assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(got))


@pytest.mark.parametrize("between", ["nothing", "quantiser", "balance"])
def test_logits_of_a_product_reach_the_layer_behind_it(between):
    """The layer's planner reads its router logits early: a product that writes them, and whatever is
    called between the two, must have let it start no sooner than the logits are there."""
    from npu_offload_b200 import MoEDataPlane
    H, F, E, K, T, KR = 512, 256, 64, 4, 2, 16384
    p, g = MoEDataPlane(H, F, E, K, n_layers=1, max_tokens=16), gen(91)
    try:
        for e in range(E):
            p.load_expert(0, e, *((randn(g, *sh) * 0.05).to(torch.bfloat16) for sh in ((F, H), (F, H), (H, F))))
        x = randn(g, T, H).to(torch.bfloat16)
        router = p.quantize_fp8(randn(g, E, KR) * KR ** -0.5, block_rows=128)
        feats = [p.quantize_fp8(randn(g, T, KR)) for _ in range(6)]
        side, logits = randn(g, 64, 4096), torch.zeros(T, E, device="cuda")
        side_logits = randn(g, 4096, E)
        side_idx = side_logits.topk(K).indices.to(torch.int32)

        def step(f, sync):
            p.matmul_fp8(f, router, out=logits)
            if sync:
                torch.cuda.synchronize()
            if between == "quantiser":
                p.quantize_fp8(side)
            elif between == "balance":
                p.balance_loss(side_logits, side_idx)
            if sync:
                torch.cuda.synchronize()
            return p.forward(0, x, logits)

        want = [step(f, True) for f in feats]
        torch.cuda.synchronize()
        assert not torch.equal(want[0], want[1])
        got = [step(f, False) for f in feats * 20]
        torch.cuda.synchronize()
        # the plan may cut the sums elsewhere behind a running call: the same experts, not the same order of sums
        for i, o in enumerate(got):
            v = want[i % len(feats)]
            assert float((o - v).abs().max()) <= 1e-4 * float(v.abs().max())
        assert p.status() == 0
    finally:
        p.close()


def test_a_wait_that_runs_out_is_reported_and_the_context_stays_usable():
    """The test hook makes the kernels wait for an arrival that nothing makes: they give up and return."""
    from npu_offload_b200 import Fp8, MoEDataPlane
    from npu_offload_b200._lib import MOE_ETIMEOUT, MOE_OK, MOE_OPT_INJECT_WAIT_TIMEOUT, MOE_OPT_WAIT_TIMEOUT_US
    g = gen(5)
    with MoEDataPlane(512, 256, 8, 2, n_layers=1, max_tokens=16) as p:
        p.set_option(MOE_OPT_WAIT_TIMEOUT_US, 2000)
        w = Fp8(*weight(g, 1500, 2048))
        xs = [p.quantize_fp8(randn(g, M, 2048)) for M in (1, 20, 40, 300)]
        calls = [lambda x=x: p.matmul_fp8(x, w) for x in xs]
        for T in (2, 20, 400):
            x, gu, d, idx, ws = expert_case(T, T, 512, 256, 8, 2)
            calls.append(lambda a=(x, Fp8(*gu), Fp8(*d), idx, ws): p.experts_fp8(*a))
        want = [c() for c in calls]
        assert p.status() == MOE_OK
        for c, v in zip(calls, want):
            p.set_option(MOE_OPT_INJECT_WAIT_TIMEOUT, 1)
            c()
            assert p.status() == MOE_ETIMEOUT
            p.set_option(MOE_OPT_INJECT_WAIT_TIMEOUT, 0)
            assert torch.equal(c(), v) and p.status() == MOE_OK


def test_a_closed_plane_refuses():
    from npu_offload_b200 import MoEDataPlane
    from npu_offload_b200._lib import MoEError
    p = MoEDataPlane(256, 64, 8, 2, n_layers=1, max_tokens=16)
    x = torch.zeros(2, 32, device="cuda")
    p.quantize_fp8(x)
    p.close()
    with pytest.raises(MoEError, match="null context"):
        p.quantize_fp8(x)


def test_calls_of_several_threads(planes):
    """Calls that share a plane, each thread on a stream of its own."""
    import threading
    from npu_offload_b200 import Fp8
    p = planes(512, 256, 16, 4)
    cases = [expert_case(40 + i, 3 + 90 * i, 512, 256, 16, 4) for i in range(3)]
    args = [(x, Fp8(*gu), Fp8(*d), idx, w) for x, gu, d, idx, w in cases]
    want = [p.experts_fp8(*a) for a in args]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(20):
            o = p.experts_fp8(*args[i], stream=s)
            s.synchronize()
            if not torch.equal(o, want[i]):
                bad.append(i)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad and p.status() == 0
