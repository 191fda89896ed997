"""64-bit definitions of the e4m3 operators and the balance loss, on any device (numpy-free torch)."""
import torch

F8 = torch.float8_e4m3fn
EPS = 2.0 ** -24  # half a step of fp32, relative


def ceil128(n):
    return -(-n // 128)


def quantize64(x, block_rows):
    """(q as 64-bit values, scale 64-bit): the definition, by comparison of exact quantities."""
    x = x.double()
    R, C = x.shape[-2:]
    rb, cb = -(-R // block_rows), ceil128(C)
    full = x.new_zeros(*x.shape[:-2], rb * block_rows, cb * 128)
    full[..., :R, :C] = x
    finite = torch.where(full.isfinite(), full.abs(), 0.0)
    top = finite.unflatten(-1, (cb, 128)).amax(-1).unflatten(-2, (rb, block_rows)).amax(-2)
    m, e = torch.frexp(top / 448)  # 2^(e-1) <= top / 448 < 2^e, exact up to the quotient's rounding
    scale = torch.ldexp(torch.ones_like(top), (e - 2).clamp(min=-126))
    for _ in range(4):
        scale = torch.where(top > 448 * scale, 2 * scale, scale)
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    v = full / expand(scale, full.shape, block_rows)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    q = torch.round(v / step) * step
    q = torch.where(full.isfinite(), q, torch.nan)
    return q[..., :R, :C], scale


def expand(scale, shape, block_rows):
    rows = torch.arange(shape[-2], device=scale.device) // block_rows
    cols = torch.arange(shape[-1], device=scale.device) // 128
    return scale.double()[..., rows, :][..., cols]


def values64(q, scale, block_rows):
    return q.double() * expand(scale, q.shape, block_rows)


def weight(g, *shape, dev="cuda", general=True, spread=0.02):
    """e4m3 weight and fp32 scales (general: not powers of two)."""
    x = torch.randn(*shape, generator=g, device=dev) * spread
    _, s = quantize64(x, 128)
    if general:
        s = s * (0.75 + 0.5 * torch.rand(s.shape, generator=g, device=dev).double())
    s = s.float()
    q = (x.double() / expand(s, x.shape, 128)).clamp(-448, 448).float().to(F8)
    return q, s.contiguous()


def matmul64(x, xs, w, ws):
    """(x . w^T, sum of |products|)"""
    a, b = values64(x, xs, 1), values64(w, ws, 128)
    return a @ b.T, a.abs() @ b.abs().T


def matmul_bound(mag, K):
    """fp32 sums in any order, products of operand and scale rounded: (K + 4) half steps of the sum of magnitudes."""
    return (K + 4) * EPS * mag


def experts64(x, gu, gus, d, ds, idx, w):
    """(out, bound): 64-bit definition, and how far fp32 sums may put the result from it.

    A sum's rounding moves an activation a by at most da; where a lies that near to a border between two
    e4m3 values it may go to the other one, a whole step away; where the group's maximum lies that near to
    a change of scale, values at the bottom of the range are rounded to twice the step."""
    T, H = x.shape
    F = d.shape[-1]
    xq = values64(*quantize64(x, 1), 1)
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    for t in range(T):
        for k in range(idx.shape[1]):
            e = int(idx[t, k])
            if e < 0:
                continue
            wg = values64(gu[e], gus[e], 128)
            g, u = wg[0] @ xq[t], wg[1] @ xq[t]
            eg, eu = (matmul_bound(wg[i].abs() @ xq[t].abs(), H) for i in (0, 1))
            sg = torch.sigmoid(g)
            a = g * sg * u
            # |d silu| <= 1.1; the fp32 expression itself: exp (2 ulp), sum, quotient, product
            da = 1.1 * eg * (u.abs() + eu) + (g * sg).abs() * eu + 8 * EPS * a.abs()
            q, s = quantize64(a[None], 1)
            se = expand(s, (1, F), 1)[0]
            v = (a / se)
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
            frac = (v / step) - torch.floor(v / step)
            near = (frac - 0.5).abs() * step * se <= da
            move = torch.where(near, step * se, 0.0)
            for b in range(ceil128(F)):
                grp = slice(128 * b, min(F, 128 * b + 128))
                top, sc = a[grp].abs().amax(), s[0, b]
                if (448 * sc - top) <= da[grp].max() or (top - 224 * sc).abs() <= da[grp].max():
                    move[grp] = torch.maximum(move[grp], 2.0 ** -8 * sc)
            wd = values64(d[e], ds[e], 128)
            aq = values64(q, s, 1)[0]
            c = float(w[t, k])
            y = wd @ aq
            out[t] += c * y
            bound[t] += abs(c) * (wd.abs() @ move + matmul_bound(wd.abs() @ (aq.abs() + move), F) + 20 * EPS * y.abs())
    return out, bound


def balance64(logits, idx, offsets, mask, scoring, grad=1.0):
    """(loss, counts [B, E], dlogits) of the definition."""
    l = logits.double()
    T, E = l.shape
    K = idx.shape[1]
    cuts = [0, T] if offsets is None else offsets.tolist()
    if scoring == "softmax":
        p = torch.softmax(l, -1)
        s = S = None
    else:
        s = torch.sigmoid(l)
        S = s.sum(-1, keepdim=True) + 1e-20
        p = s / S
    keep = torch.ones(T, dtype=torch.bool, device=l.device) if mask is None else mask.bool()
    spans = [torch.nonzero(keep[a:b])[:, 0] + a for a, b in zip(cuts[:-1], cuts[1:])]
    full = sum(len(t) > 0 for t in spans)
    loss, d, counts = l.new_zeros(()), torch.zeros_like(l), []
    for t in spans:
        ch = idx[t].reshape(-1).long()
        c = torch.bincount(ch[ch >= 0], minlength=E)
        counts.append(c)
        if len(t):
            f = c.double() * E / (K * len(t))
            loss = loss + (f * p[t].mean(0)).sum() / full
            g = grad * f / (len(t) * full)
            dp = g - (g * p[t]).sum(-1, keepdim=True)
            d[t] = p[t] * dp if s is None else s[t] * (1 - s[t]) / S[t] * dp
    return loss, torch.stack(counts).int(), d
