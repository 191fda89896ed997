"""What is measured of the 8-bit floating-point path and the router's balance loss.

quantize   rows (or 128 x 128 blocks) of a matrix to e4m3 with one scale for each 128 values
matmul     out = x . w^T on e4m3 operands, x scaled per row and 128 columns, w per 128 x 128 block
experts    the routed SwiGLU experts of one MoE layer on e4m3 weights: quantised tokens, gate and up
           product, SwiGLU, quantised activations, down product, weighted sum over each token's experts
balance    the router's load-balance loss with the per-expert counts, and its gradient

A case's sizes are the MoE layer's own (hidden 4096, intermediate 1280, 128 experts, 8 per token) or generic.
"""
import math

import torch

own = False

BLOCK = 128          # values (or rows and columns) under one scale
E4M3_MAX = 448.0
F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one token's hidden state on its way into a product
        dict(name="quantize token", op="quantize", rows=1, cols=4096, block_rows=1, dtype="bf16"),
        # SwiGLU activations of a ragged prompt, fp32
        dict(name="quantize rows fp32", op="quantize", rows=8191, cols=1280, block_rows=1, dtype="fp32"),
        # weight matrices on their way into 8 bits: gate and up rows of sixteen experts
        dict(name="quantize weights", op="quantize", rows=40960, cols=4096, block_rows=128, dtype="bf16"),
        # the shared expert's gate and up rows for one token
        dict(name="matmul token", op="matmul", M=1, N=2560, K=4096, out="bf16"),
        # its down product for a handful of tokens, into fp32
        dict(name="matmul 13 tokens", op="matmul", M=13, N=4096, K=1280, out="fp32"),
        # a ragged prompt
        dict(name="matmul prompt", op="matmul", M=517, N=2560, K=4096, out="bf16"),
        # a large square product
        dict(name="matmul large", op="matmul", M=8192, N=8192, K=8192, out="bf16"),
        # one token through its 8 of 128 experts
        dict(name="experts token", op="experts", T=1, H=4096, F=1280, E=128, K=8, zipf=True, out="bf16"),
        # a decode batch with popular and rare experts
        dict(name="experts batch", op="experts", T=16, H=4096, F=1280, E=128, K=8, zipf=True, out="bf16"),
        # a prompt, about 128 tokens an expert
        dict(name="experts prompt", op="experts", T=2048, H=4096, F=1280, E=128, K=8, zipf=False, out="bf16"),
        # ragged sequences (one of them empty) with padded tokens, sigmoid scores
        dict(name="balance ragged", op="balance", T=4090, E=128, K=8, B=9, masked=True, scoring="sigmoid"),
        # a training batch
        dict(name="balance batch", op="balance", T=65536, E=256, K=8, B=1, masked=False, scoring="softmax"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "experts", "experts", "balance"])
    if op == "quantize":
        block = rng.choice([1, 1, 128])
        cols = 16 * _log(rng, 1, 640)
        rows = _log(rng, 1, min(32768, 160_000_000 // cols))
        return dict(op=op, rows=rows, cols=cols, block_rows=block, dtype=rng.choice(["bf16", "fp32"]))
    if op == "matmul":
        return dict(op=op, M=_log(rng, 1, 8192), N=_log(rng, 16, 8192), K=16 * _log(rng, 4, 512), out=rng.choice(["bf16", "fp32"]))
    if op == "experts":
        K = rng.choice([1, 2, 4, 6, 8])
        return dict(op=op, T=_log(rng, 1, 2048), H=64 * _log(rng, 4, 64), F=64 * _log(rng, 1, 20), E=rng.choice([8, 16, 60, 64, 128]), K=K,
                    zipf=rng.choice([True, False]), out="bf16")
    E = rng.choice([8, 16, 60, 64, 128, 160, 256])
    return dict(op=op, T=_log(rng, 1, 65536), E=E, K=rng.choice([1, 2, 4, 6, 8]), B=rng.choice([1, 1, 3, 17, 64]), masked=rng.choice([True, False]),
                scoring=rng.choice(["softmax", "sigmoid"]))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _blocks(x, block_rows):
    """x [..., R, C] padded with zeros and cut: [..., row blocks, block_rows, column blocks, 128]."""
    R, C = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -C % BLOCK, 0, -R % block_rows))
    return x.reshape(*x.shape[:-2], -1, block_rows, x.shape[-1] // BLOCK, BLOCK)


def _checkpoint_weight(g, *shape):
    """An e4m3 weight as a checkpoint holds it: N(0, 0.02), one fp32 scale (largest value / 448) for each 128 x 128 block."""
    b = _blocks(_randn(g, *shape) * 0.02, BLOCK)
    s = b.abs().amax((-3, -1)) / E4M3_MAX
    q = (b / s[..., :, None, :, None]).to(F8)
    q = q.reshape(*shape[:-2], b.shape[-4] * BLOCK, b.shape[-2] * BLOCK)[..., : shape[-2], : shape[-1]]
    return q.contiguous(), s.contiguous()


def _expert_weights(g, E, rest):
    """Weights of E experts, made a few at a time."""
    parts = [_checkpoint_weight(g, n, *rest) for n in [16] * (E // 16) + ([E % 16] if E % 16 else [])]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def _logits(g, T, E, zipf):
    x = _randn(g, T, E)
    if zipf:
        x = x - torch.log(torch.randperm(E, generator=g, device="cuda").float() + 1)
    return x


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
    if case["op"] == "quantize":
        x = _randn(g, case["rows"], case["cols"])
        x *= 0.02 if case["block_rows"] == 128 else torch.exp(_randn(g, case["rows"], 1))
        s["x"] = x.to(torch.bfloat16) if case["dtype"] == "bf16" else x
        config = dict(hidden=256, inter=64, n_experts=8, top_k=2)
    elif case["op"] == "matmul":
        x = _blocks(_randn(g, case["M"], case["K"]), 1)
        scale = _power_of_two_scale(x.abs().amax((-3, -1)))
        q = (x / scale[:, None, :, None]).to(F8).reshape(case["M"], -1)[:, : case["K"]].contiguous()
        s["x"], s["w"] = (q, scale.contiguous()), _checkpoint_weight(g, case["N"], case["K"])
        config = dict(hidden=256, inter=64, n_experts=8, top_k=2)
    elif case["op"] == "experts":
        T, H, F, E, K = (case[k] for k in "THFEK")
        s["gate_up"], s["down"] = _expert_weights(g, E, (2, F, H)), _expert_weights(g, E, (H, F))
        s["x"] = _randn(g, T, H).to(torch.bfloat16)
        p, idx = torch.softmax(_logits(g, T, E, case["zipf"]), -1).topk(K, -1)
        s["idx"], s["weights"] = idx.to(torch.int32), p / p.sum(-1, keepdim=True)
        config = dict(hidden=H, inter=F, n_experts=E, top_k=K)
    else:
        T, E, K, B = (case[k] for k in "TEKB")
        s["logits"] = _logits(g, T, E, True)
        s["idx"] = s["logits"].topk(K, -1)[1].to(torch.int32)
        cuts = torch.rand(B - 1, generator=g, device="cuda").mul(T).long().sort()[0]
        if B > 2:
            cuts[1] = cuts[0]  # an empty sequence
        ends = torch.tensor([0, T], device="cuda")
        s["offsets"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32) if B > 1 else None
        s["mask"] = torch.rand(T, generator=g, device="cuda") > 0.1 if case["masked"] else None
        s["grad"] = torch.full((), 0.01, device="cuda") * (1 + torch.rand((), generator=g, device="cuda"))
        config = dict(hidden=256, inter=64, n_experts=E, top_k=K, scoring=case["scoring"])
    if own:
        from npu_offload_b200 import Fp8
        s["plane"] = _plane(**config)
        for name in ("w", "gate_up", "down"):
            if name in s:
                s[name] = Fp8(*s[name])
        if case["op"] == "matmul":
            s["x"] = Fp8(*s["x"])
    return s


# ---------------------------------------------------------------- plain forms

def _power_of_two_scale(largest):
    """The smallest power of two s with largest <= 448 s (at least 2^-126); 1 where there is nothing but zeros."""
    m, e = torch.frexp(largest)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), e), 1.0)


def _quantize(x, block_rows):
    """(e4m3 values, scales): infinities and NaN become NaN and count for no scale."""
    b = _blocks(x.float(), block_rows)
    scale = _power_of_two_scale(torch.where(b.isfinite(), b.abs(), 0).amax((-3, -1)))
    q = (b / scale[..., :, None, :, None]).to(F8)
    q = q.reshape(*x.shape[:-2], b.shape[-4] * block_rows, -1)[..., : x.shape[-2], : x.shape[-1]]
    return q.contiguous(), scale


def _dequant(q, scale, block_rows):
    s = scale.repeat_interleave(block_rows, -2) if block_rows > 1 else scale
    return q.float() * s[..., : q.shape[-2], :].repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]


def _matmul(x, w, out):
    y = _dequant(*x, 1) @ _dequant(*w, BLOCK).T
    return y.to(torch.bfloat16) if out == "bf16" else y


def _swiglu(gate_up):
    gate, up = gate_up
    return gate / (1 + torch.exp(-gate)) * up


def _experts(s):
    T, F, E, K = (s[k] for k in "TFEK")
    x = _dequant(*_quantize(s["x"], 1), 1)
    pairs = s["idx"].reshape(-1).long()
    if T * K < E:  # few pairs: their experts alone
        of = lambda w: _dequant(w[0][pairs], w[1][pairs], BLOCK)  # noqa: E731
        rows = x.repeat_interleave(K, 0)[:, None]
    else:  # the tokens of each expert, filled up to the longest list
        of = lambda w: _dequant(*w, BLOCK)  # noqa: E731
        order = pairs.argsort(stable=True)
        count = torch.bincount(pairs, minlength=E)
        place = torch.arange(T * K, device=x.device) - (count.cumsum(0) - count)[pairs[order]]
        rows = x.new_zeros(E, int(count.max()), x.shape[1])
        rows[pairs[order], place] = x[order // K]
    gate_up = torch.einsum("nth,ngfh->gntf", rows, of(s["gate_up"]))
    act = _dequant(*_quantize(_swiglu(gate_up), 1), 1)
    y = torch.einsum("ntf,nhf->nth", act, of(s["down"]))
    if T * K < E:
        y = y[:, 0]
    else:
        y = torch.empty(T * K, x.shape[1], device=x.device).index_copy(0, order, y[pairs[order], place])
    return (y.reshape(T, K, -1) * s["weights"][:, :, None]).sum(1).to(torch.bfloat16)


def _balance(s):
    E, K, logits = s["E"], s["K"], s["logits"]
    T, dev = logits.shape[0], logits.device
    offsets = torch.tensor([0, T], device=dev) if s["offsets"] is None else s["offsets"].long()
    at = torch.arange(T, device=dev)
    member = (at >= offsets[:-1, None]) & (at < offsets[1:, None])  # [B, T]
    if s["mask"] is not None:
        member = member & s["mask"]
    member = member.float()
    chosen = (s["idx"][:, :, None] == torch.arange(E, device=dev)).sum(1).float()
    if s["scoring"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        total = e.sum(-1, keepdim=True)
    else:
        e = 1 / (1 + torch.exp(-logits))
        total = e.sum(-1, keepdim=True) + 1e-20
    p = e / total
    n = member.sum(-1, keepdim=True)
    counts = member @ chosen
    share = torch.where(n > 0, E / K * counts / n.clamp(min=1), 0)
    mean = torch.where(n > 0, member @ p / n.clamp(min=1), 0)
    sequences = (n > 0).sum().clamp(min=1)
    loss = (share * mean).sum() / sequences
    # the gradient: share and counts are constants, p is not
    f = member.T @ (share / n.clamp(min=1)) * (s["grad"] / sequences)  # [T, E], 0 for tokens of no sequence
    inner = (f * p).sum(-1, keepdim=True)
    slope = p if s["scoring"] == "softmax" else e * (1 - e) / total
    return loss, counts.to(torch.int32), slope * (f - inner)


def run(s):
    if s["op"] == "quantize":
        return tuple(s["plane"].quantize_fp8(s["x"], block_rows=s["block_rows"])) if own else _quantize(s["x"], s["block_rows"])
    if s["op"] == "matmul":
        if own:
            return s["plane"].matmul_fp8(s["x"], s["w"], out_dtype=torch.bfloat16 if s["out"] == "bf16" else torch.float32)
        return _matmul(s["x"], s["w"], s["out"])
    if s["op"] == "experts":
        if own:
            return s["plane"].experts_fp8(s["x"], s["gate_up"], s["down"], s["idx"], s["weights"], out_dtype=torch.bfloat16)
        return _experts(s)
    if own:
        loss, stats = s["plane"].balance_loss(s["logits"], s["idx"], offsets=s["offsets"], mask=s["mask"])
        return loss, stats.counts, s["plane"].balance_loss_backward(s["logits"], stats, s["grad"])
    return _balance(s)


# ---------------------------------------------------------------- work

def _ceil(a, b):
    return -(-a // b)


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        scales = _ceil(case["rows"], case["block_rows"]) * _ceil(case["cols"], BLOCK)
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + n + 4 * scales, "flops": 3 * n}
    if case["op"] == "matmul":
        M, N, K = (case[k] for k in "MNK")
        kb = _ceil(K, BLOCK)
        return {"bytes": M * K + N * K + 4 * kb * (M + _ceil(N, BLOCK)) + M * N * (2 if case["out"] == "bf16" else 4), "flops": 2 * M * N * K}
    if case["op"] == "experts":
        T, H, F, E, K = (case[k] for k in "THFEK")
        popular = [1 / (i + 1) if case["zipf"] else 1.0 for i in range(E)]
        total = sum(popular)
        # experts that T tokens reach: each of a token's K choices taken for an independent draw
        reached = E if K >= E else min(sum(1 - (1 - p / total) ** (T * K) for p in popular) if T > 1 else K, E)
        scales = 4 * 3 * _ceil(F, BLOCK) * _ceil(H, BLOCK)
        return {"bytes": reached * (3 * F * H + scales) + T * H * (2 + 2) + T * K * 8, "flops": 6 * T * K * F * H}
    T, E, K, B = (case[k] for k in "TEKB")
    # logits for the loss and again for its gradient, which needs every token's sums first
    return {"bytes": T * E * 4 * 3 + T * K * 4 + (T if case["masked"] else 0) + 4 * B * (E + 1), "flops": 12 * T * E}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_quantize(x, block_rows):
    R, C = x.shape[-2:]
    rb, cb = _ceil(R, block_rows), _ceil(C, BLOCK)
    full = torch.zeros(*x.shape[:-2], rb * block_rows, cb * BLOCK, dtype=torch.float64, device=x.device)
    full[..., :R, :C] = x.double()
    top = full.unflatten(-1, (cb, BLOCK)).abs().amax(-1).unflatten(-2, (rb, block_rows)).amax(-2)
    scale = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-126))
    # log2 may round across a power of two: put it right by comparison
    scale = torch.where(top > 448 * scale, 2 * scale, torch.where((top <= 224 * scale) & (scale > 2.0 ** -126), scale / 2, scale))
    scale[top == 0] = 1
    value = full / scale.repeat_interleave(block_rows, -2).repeat_interleave(BLOCK, -1)
    # three bits behind the leading one, down to steps of 2^-9; ties to even
    step = torch.exp2(torch.floor(torch.log2(value.abs().clamp(min=2.0 ** -20))).clamp(min=-6) - 3)
    return (torch.round(value / step) * step)[..., :R, :C], scale


def _exact_values(q, scale, block_rows):
    rows = torch.arange(q.shape[-2], device=q.device) // block_rows
    cols = torch.arange(q.shape[-1], device=q.device) // BLOCK
    return q.double() * scale.double()[..., rows, :][..., cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_quantize(s["x"], case["block_rows"])
    if case["op"] == "matmul":
        return _exact_values(*s["x"], 1).matmul(_exact_values(*s["w"], BLOCK).transpose(0, 1))
    if case["op"] == "experts":
        q, scale = _exact_quantize(s["x"], 1)
        x = _exact_values(q, scale, 1)
        out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
        for e in torch.unique(s["idx"]).tolist():
            token, k = torch.nonzero(s["idx"] == e, as_tuple=True)
            w = _exact_values(s["gate_up"][0][e], s["gate_up"][1][e], BLOCK)
            gate, up = x[token] @ w[0].T, x[token] @ w[1].T
            q, scale = _exact_quantize(gate * torch.sigmoid(gate) * up, 1)
            y = _exact_values(q, scale, 1) @ _exact_values(s["down"][0][e], s["down"][1][e], BLOCK).T
            out[token] += s["weights"][token, k, None].double() * y
        return out
    T, E, K = (case[k] for k in "TEK")
    logits = s["logits"].double()
    cuts = [0, T] if s["offsets"] is None else s["offsets"].tolist()
    score = torch.softmax(logits, -1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    total = 1.0 if case["scoring"] == "softmax" else score.sum(-1, keepdim=True) + 1e-20
    p = score / total
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    spans = [torch.nonzero(keep[a:b])[:, 0] + a for a, b in zip(cuts[:-1], cuts[1:])]
    full = sum(len(t) > 0 for t in spans)
    loss, counts, grad = 0.0, [], torch.zeros_like(logits)
    for t in spans:
        c = torch.bincount(s["idx"][t].reshape(-1).long(), minlength=E)
        counts.append(c)
        if len(t):
            f = c.double() * E / (K * len(t))
            loss += float((f * p[t].mean(0)).sum()) / full
            g = s["grad"].double() * f / (len(t) * full)
            dp = g - (g * p[t]).sum(-1, keepdim=True)
            grad[t] = p[t] * dp if case["scoring"] == "softmax" else score[t] * (1 - score[t]) / total[t] * dp
    return torch.tensor(loss, dtype=torch.float64), torch.stack(counts).to(torch.int32), grad
