"""What is measured of the steps around the routed experts: norm, routing in groups, adapters.

norm            residual addition and root-mean-square norm, to bf16 / fp32 and / or e4m3 with one scale for each 128 values
norm_backward   its gradients: of the sum (so of x and of the residual) and of the weight
route           top-k routing limited to the best groups of experts
route_backward  the gradient of the routing weights, to the logits
lora            low-rank adapters of many requests beside a shared projection

A case's sizes are the MoE layer's own (hidden 4096, intermediate 1280, 128 experts, 8 per token) or generic.
"""
import math

import torch

own = False

BLOCK = 128  # values under one scale
E4M3_MAX = 448.0
F8 = torch.float8_e4m3fn
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # the experts' fp32 sums of one decoded token into the next block: bf16 for its router, e4m3 for its products
        dict(name="norm token", op="norm", T=1, C=4096, x="fp32", residual="bf16", out="bf16", fp8=True),
        # a ragged prompt on its way into e4m3 products alone
        dict(name="norm prompt", op="norm", T=2047, C=4096, x="bf16", residual="bf16", out="none", fp8=True),
        # a training batch
        dict(name="norm batch", op="norm", T=16384, C=4096, x="bf16", residual="bf16", out="bf16", fp8=False),
        # a small step on an fp32 stream, the last norm of a model: nothing else flows into its input
        dict(name="norm gradient small", op="norm_backward", T=517, C=1280, sum="fp32", dy="fp32", dsum=False),
        # a training batch, with the gradient that comes down the residual stream
        dict(name="norm gradient batch", op="norm_backward", T=8191, C=4096, sum="bf16", dy="bf16", dsum=True),
        # one decoded token, sigmoid scores with a balance bias
        dict(name="route token", op="route", T=1, E=128, K=8, G=8, top=3, scoring="sigmoid", renormalize=True, scale=2.5),
        # a training batch of the widest router
        dict(name="route batch", op="route", T=65536, E=256, K=8, G=8, top=4, scoring="sigmoid", renormalize=True, scale=2.5),
        # a ragged batch, probabilities as they are
        dict(name="route gradient ragged", op="route_backward", T=4090, E=160, K=6, scoring="softmax", renormalize=False, scale=16.0),
        # a training batch
        dict(name="route gradient batch", op="route_backward", T=65536, E=256, K=8, scoring="sigmoid", renormalize=True, scale=2.5),
        # one decoded token of one request, beside the shared expert's gate and up rows
        dict(name="lora token", op="lora", T=1, K=4096, N=2560, r=16, n=8, runs=False, out="bf16"),
        # a decode batch of requests with adapters of their own, beside the shared expert's down rows, into fp32
        dict(name="lora batch", op="lora", T=48, K=1280, N=4096, r=32, n=32, runs=False, out="fp32"),
        # prompts of several requests, some without an adapter
        dict(name="lora prompts", op="lora", T=4093, K=4096, N=2560, r=16, n=16, runs=True, out="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "route", "route_backward", "lora", "lora"])
    if op == "norm":
        fp8 = rng.choice([True, False])
        C = 16 * _log(rng, 1, 512) if fp8 else _log(rng, 1, 8192)
        return dict(op=op, T=_log(rng, 1, min(16384, 67_000_000 // C)), C=C, x=rng.choice(["bf16", "fp32"]),
                    residual=rng.choice(["bf16", "fp32", "none"]), out=rng.choice(["bf16", "fp32"] + ["none"] * fp8), fp8=fp8)
    if op == "norm_backward":
        C = _log(rng, 8, 8192)  # (one channel's gradient is what rounding leaves of a difference)
        return dict(op=op, T=_log(rng, 1, min(8192, 33_000_000 // C)), C=C, sum=rng.choice(["bf16", "fp32"]),
                    dy=rng.choice(["bf16", "fp32"]), dsum=rng.choice([True, False]))
    scoring, renormalize, scale = rng.choice(["softmax", "sigmoid"]), rng.choice([True, False]), rng.choice([1.0, 2.5])
    if op == "route":
        G, per = rng.choice([(1, 8), (1, 60), (1, 256), (3, 20), (4, 16), (4, 32), (8, 8), (8, 16), (8, 20), (8, 32), (16, 16)])
        top = rng.randint(1, G)
        K = rng.randint(1, min(16, top * per))
        return dict(op=op, T=_log(rng, 1, 65536), E=G * per, K=K, G=G, top=top, scoring=scoring, renormalize=renormalize, scale=scale)
    if op == "route_backward":
        E = rng.choice([8, 16, 60, 64, 128, 160, 256])
        K = rng.choice([2, 4, 6, 8] if renormalize else [1, 2, 4, 6, 8])  # (a lone renormalised weight has no gradient)
        return dict(op=op, T=_log(rng, 1, 65536), E=E, K=K, scoring=scoring, renormalize=renormalize, scale=scale)
    return dict(op=op, T=_log(rng, 1, 4096), K=8 * _log(rng, 8, 512), N=8 * _log(rng, 2, 320), r=rng.choice([8, 16, 24, 32, 64]),
                n=rng.choice([1, 4, 16, 32]), runs=rng.choice([True, False]), out=rng.choice(["bf16", "fp32"]))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stream(g, T, C):
    """A residual stream's values: tokens of unlike size, a few channels that stand out."""
    return _randn(g, T, C) * torch.exp(0.5 * _randn(g, T, 1)) * torch.exp(0.7 * _randn(g, C))


_planes = {}


def _plane(**config):
    """The data plane that a program keeps: its limits, device and error state."""
    from npu_offload_b200 import MoEDataPlane
    key = tuple(sorted(config.items()))
    if key not in _planes:
        _planes[key] = MoEDataPlane(max_tokens=16, **config)
    return _planes[key]


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    config = dict(hidden=256, inter=64, n_experts=8, top_k=2)
    if case["op"] == "norm":
        T, C = case["T"], case["C"]
        s["x_"] = _stream(g, T, C).to(TYPES[case["x"]])
        s["residual_"] = _stream(g, T, C).to(TYPES[case["residual"]]) if case["residual"] != "none" else None
        s["weight"] = (1 + 0.2 * _randn(g, C)).to(torch.bfloat16)
    elif case["op"] == "norm_backward":
        T, C = case["T"], case["C"]
        s["sum_"] = _stream(g, T, C).to(TYPES[case["sum"]])
        s["weight"] = (1 + 0.2 * _randn(g, C)).to(torch.bfloat16)
        s["dy_"] = (1e-3 * _randn(g, T, C)).to(TYPES[case["dy"]])
        s["dsum_"] = (1e-3 * _randn(g, T, C)).to(TYPES[case["sum"]]) if case["dsum"] else None
        s["rstd"] = torch.rsqrt(s["sum_"].double().square().mean(-1) + EPS).float()
    elif case["op"] == "lora":
        T, K, N, r, n = (case[k] for k in ("T", "K", "N", "r", "n"))
        s["x"] = _randn(g, T, K).to(torch.bfloat16)
        s["a"] = (_randn(g, n, r, K) * K ** -0.5).to(torch.bfloat16)
        s["b"] = (_randn(g, n, N, r) * 0.1).to(torch.bfloat16)
        s["scaling"] = 0.5 + torch.rand(n, generator=g, device="cuda")
        s["base"] = _randn(g, T, N).to(TYPES[case["out"]])
        ids = torch.randint(-1 if T > 1 else 0, n, (T,), generator=g, device="cuda")
        if case["runs"]:  # requests one after the other, of unlike lengths
            starts = torch.rand(T, generator=g, device="cuda") < 0.003
            ids = ids[starts.cumsum(0)]
        s["ids"] = ids.to(torch.int32)
    else:
        T, E, K = (case[k] for k in "TEK")
        s["logits"] = _randn(g, T, E) - 0.3 * torch.log(torch.randperm(E, generator=g, device="cuda").float() + 1)
        if case["op"] == "route":
            s["bias"] = 0.05 * _randn(g, E) if case["scoring"] == "sigmoid" else None
        else:
            s["idx"] = s["logits"].topk(K, -1)[1].to(torch.int32)
            s["dw"] = 1e-3 * _randn(g, T, K)
        config = dict(hidden=256, inter=64, n_experts=E, top_k=K, scoring=case["scoring"])
    if own:
        s["plane"] = _plane(**config)
    return s


# ---------------------------------------------------------------- plain forms

def _power_of_two_scale(largest):
    """The smallest power of two s with largest <= 448 s (at least 2^-126); 1 where there is nothing but zeros."""
    m, e = torch.frexp(largest)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), e), 1.0)


def _norm(s):
    x, residual, w = s["x_"], s["residual_"], s["weight"]
    h = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    rstd = torch.rsqrt(h.float().square().mean(-1) + EPS)
    v = h.float() * rstd[:, None] * w.float()
    y = q = scale = None
    if s["out"] != "none":
        y = v.to(TYPES[s["out"]])
    if s["fp8"]:  # a scale doubles at a border: in 64 bits
        h64 = h.double()
        v64 = h64 * torch.rsqrt(h64.square().mean(-1, keepdim=True) + EPS) * w.double()
        pad = (0, -s["C"] % BLOCK)
        scale = _power_of_two_scale(torch.nn.functional.pad(v64.abs(), pad).unflatten(-1, (-1, BLOCK)).amax(-1)).float()
        q = torch.nn.functional.pad(v, pad).unflatten(-1, (-1, BLOCK)) / scale[..., None]
        q = q.to(F8).flatten(1)[:, : s["C"]].contiguous()
    return y, q, scale, None if residual is None else h, rstd


def _norm_backward(s):
    h, dy, rstd = s["sum_"].float(), s["dy_"].float(), s["rstd"][:, None]
    unit = h * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    if s["dsum_"] is not None:
        dx = dx + s["dsum_"].float()
    return dx.to(s["sum_"].dtype), (dy * unit).sum(0)


def _sigmoid(logits):
    """With the exponential rounded once, as the router's other calls form it."""
    return 1 / (1 + torch.exp(-logits.double()).float())


def _route(s):
    logits, E, K, G = s["logits"], s["E"], s["K"], s["G"]
    T = logits.shape[0]
    if s["scoring"] == "softmax":
        key = logits
        group = key.view(T, G, -1).amax(-1)
    else:
        score = _sigmoid(logits)
        key = score + s["bias"]
        group = key.view(T, G, -1).sort(dim=-1, descending=True)[0][..., :2].sum(-1)
    best = group.sort(dim=-1, descending=True, stable=True)[1][:, : s["top"]]
    open_ = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter(1, best, True)
    open_ = open_[:, :, None].expand(T, G, E // G).reshape(T, E)
    idx = torch.where(open_, key, -math.inf).sort(dim=-1, descending=True, stable=True)[1][:, :K]
    if s["scoring"] == "softmax":
        v = torch.exp(logits - logits.amax(-1, keepdim=True))
        v = v / v.sum(-1, keepdim=True)
    else:
        v = score
    w = v.gather(-1, idx)
    if s["renormalize"]:
        w = w / (w.sum(-1, keepdim=True) + (1e-20 if s["scoring"] == "sigmoid" else 0))
    return idx.to(torch.int32), w * s["scale"]


def _route_backward(s):
    logits, idx, g = s["logits"], s["idx"].long(), s["dw"] * s["scale"]
    if s["scoring"] == "softmax":
        v = torch.exp(logits - logits.amax(-1, keepdim=True))
        v = v / v.sum(-1, keepdim=True)
    else:
        v = 1 / (1 + torch.exp(-logits))
    if s["renormalize"]:
        chosen = v.gather(-1, idx)
        total = chosen.sum(-1, keepdim=True) + (1e-20 if s["scoring"] == "sigmoid" else 0)
        g = (g - (g * chosen).sum(-1, keepdim=True) / total) / total
    dv = torch.zeros_like(logits).scatter(-1, idx, g)
    if s["scoring"] == "softmax":
        return v * (dv - (dv * v).sum(-1, keepdim=True))
    return dv * v * (1 - v)


def _lora(s):
    n, r, K = s["a"].shape
    own_rows = s["ids"].long()[:, None] == torch.arange(n, device=s["ids"].device)  # [T, n]
    low = (s["x"].float() @ s["a"].float().reshape(n * r, K).T).reshape(-1, n, r)
    low = torch.where(own_rows[:, :, None], low * s["scaling"][:, None], 0)
    delta = low.reshape(-1, n * r) @ s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return (s["base"].float() + delta).to(s["base"].dtype)


def run(s):
    if s["op"] == "norm":
        if own:
            n = s["plane"].add_norm(s["x_"], s["weight"], s["residual_"], eps=EPS, out_dtype=TYPES.get(s["out"]), fp8=s["fp8"])
            q, scale = (None, None) if n.fp8 is None else n.fp8
            return n.y, q, scale, None if s["residual_"] is None else n.sum, n.rstd
        return _norm(s)
    if s["op"] == "norm_backward":
        return s["plane"].add_norm_backward(s["dy_"], s["sum_"], s["weight"], s["rstd"], dsum=s["dsum_"]) if own else _norm_backward(s)
    if s["op"] == "route":
        if own:
            return s["plane"].route_groups(s["logits"], s["G"], s["top"], bias=s["bias"], renormalize=s["renormalize"], scale=s["scale"])
        return _route(s)
    if s["op"] == "route_backward":
        if own:
            return s["plane"].route_backward(s["logits"], s["idx"], s["dw"], renormalize=s["renormalize"], scale=s["scale"])
        return _route_backward(s)
    return s["plane"].add_lora(s["base"], s["x"], s["a"], s["b"], s["ids"], scale=s["scaling"]) if own else _lora(s)


# ---------------------------------------------------------------- work

_BYTES = {"bf16": 2, "fp32": 4, "none": 0}


def work(case):
    op, T = case["op"], case["T"]
    if op == "norm":
        C, stream = case["C"], _BYTES[case["residual"]]
        each = _BYTES[case["x"]] + 2 * stream + _BYTES[case["out"]]
        return {"bytes": T * C * (each + case["fp8"]) + 2 * C + 4 * T * (1 + case["fp8"] * -(-C // BLOCK)), "flops": (5 + 2 * case["fp8"]) * T * C}
    if op == "norm_backward":
        C, stream = case["C"], _BYTES[case["sum"]]
        return {"bytes": T * C * (stream * (2 + case["dsum"]) + _BYTES[case["dy"]]) + 6 * C + 4 * T, "flops": 10 * T * C}
    if op == "lora":
        K, N, r, n = (case[k] for k in ("K", "N", "r", "n"))
        # adapters that T tokens, or the runs among them, reach; each choice one of n and of none
        choices = 1 + 0.003 * (T - 1) if case["runs"] else T
        used = 1 if T == 1 else n * (1 - (1 - 1 / (n + 1)) ** choices)
        return {"bytes": int(T * K * 2 + 2 * T * N * _BYTES[case["out"]] + used * (r * (K + N) * 2 + 4) + 4 * T), "flops": 2 * T * r * (K + N)}
    E, K = case["E"], case["K"]
    if op == "route":
        return {"bytes": T * E * 4 + T * K * 8 + 4 * E, "flops": 8 * T * E}
    # the whole row of logits where its sum is needed, else the chosen ones'
    read = E if case["scoring"] == "softmax" and not case["renormalize"] else K
    return {"bytes": 4 * T * (E + read) + T * K * 8, "flops": 6 * T * read}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_quantize(v):
    T, C = v.shape
    blocks = -(-C // BLOCK)
    top = torch.stack([v[:, i * BLOCK:(i + 1) * BLOCK].abs().amax(-1) for i in range(blocks)], -1)
    scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=-126))
    # log2 may round across a power of two: put it right by comparison
    scale = torch.where(top > E4M3_MAX * scale, 2 * scale, torch.where((top <= E4M3_MAX / 2 * scale) & (scale > 2.0 ** -126), scale / 2, scale))
    scale[top == 0] = 1
    value = v / scale[:, torch.arange(C, device=v.device) // BLOCK]
    # three bits behind the leading one, down to steps of 2^-9; ties to even
    step = torch.exp2(torch.floor(torch.log2(value.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return torch.round(value / step) * step, scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x_"].double()
        if s["residual_"] is not None:  # the sum as the stream holds it
            h = (h + s["residual_"].double()).to(s["residual_"].dtype).double()
        rstd = (h.pow(2).sum(-1) / case["C"] + EPS).pow(-0.5)
        v = torch.einsum("tc,t,c->tc", h, rstd, s["weight"].double())
        q, scale = _exact_quantize(v) if case["fp8"] else (None, None)
        return None if case["out"] == "none" else v, q, scale, None if s["residual_"] is None else h, rstd
    if case["op"] == "norm_backward":
        h, dy, w, rstd = s["sum_"].double(), s["dy_"].double(), s["weight"].double(), s["rstd"].double()
        inner = torch.einsum("tc,tc,c->t", dy, h, w) * rstd.pow(3) / case["C"]
        dx = dy * w * rstd[:, None] - h * inner[:, None]
        return dx + (0 if s["dsum_"] is None else s["dsum_"].double()), torch.einsum("tc,tc,t->c", dy, h, rstd)
    if case["op"] == "lora":
        out = s["base"].double()
        for i in torch.unique(s["ids"]).tolist():
            if i >= 0:
                t = torch.nonzero(s["ids"] == i)[:, 0]
                out[t] += float(s["scaling"][i]) * (s["x"][t].double() @ s["a"][i].double().T @ s["b"][i].double().T)
        return out
    logits = s["logits"].double()
    score = torch.softmax(logits, -1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    if case["op"] == "route":
        idx = _route(s)[0]  # a choice is defined on fp32 keys; the weights on real numbers
        w = torch.take_along_dim(score, idx.long(), -1)
        return idx, case["scale"] * (w / w.sum(-1, keepdim=True) if case["renormalize"] else w)
    at, g = s["idx"].long(), case["scale"] * s["dw"].double()
    v = torch.take_along_dim(score, at, -1)
    if case["renormalize"]:
        p = v / v.sum(-1, keepdim=True)
        # d w / d logit: of softmax among the chosen, or by the logarithms of the sigmoids
        d = p * (g - (g * p).sum(-1, keepdim=True)) * (1 if case["scoring"] == "softmax" else 1 - v)
        return torch.zeros_like(logits).scatter_add_(-1, at, d)
    if case["scoring"] == "sigmoid":
        return torch.zeros_like(logits).scatter_add_(-1, at, g * v * (1 - v))
    return torch.zeros_like(logits).scatter_add_(-1, at, g * v) - score * (g * v).sum(-1, keepdim=True)
