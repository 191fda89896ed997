"""Routing limited to groups and the weights' gradient, in plain form, for their tests."""
import numpy as np
import torch


def keys(logits, bias, scoring):
    """The fp32 numbers that choices are made by."""
    if scoring == "softmax":
        return logits.cpu().numpy() + np.float32(0)
    e = torch.exp(-logits.double()).float()  # the exponential rounded once
    s = 1 / (1 + e)
    return (s if bias is None else s + bias).cpu().numpy() + np.float32(0)


def choose(logits, groups, top, K, bias=None, scoring="softmax"):
    """idx [T, K] by sorting: larger first, ties to the lower index; NaN as -inf."""
    key = keys(logits, bias, scoring)
    key = np.where(np.isnan(key), np.float32(-np.inf), key)
    T, E = key.shape
    size = E // groups
    out = np.empty((T, K), np.int32)
    for t in range(T):
        by_group = -np.sort(-key[t].reshape(groups, size), -1)
        with np.errstate(invalid="ignore"):
            score = by_group[:, 0] if scoring == "softmax" or size == 1 else by_group[:, 0] + by_group[:, 1]
        score = np.where(np.isnan(score), np.float32(-np.inf), score)
        best = np.lexsort((np.arange(groups), -score))[:top]
        inside = [e for g in sorted(best) for e in range(g * size, (g + 1) * size)]
        inside.sort(key=lambda e: (-key[t, e], e))
        out[t] = inside[:K]
    return torch.from_numpy(out)


def weights64(logits, idx, scoring, renormalize, scale):
    l = logits.double()
    v = torch.softmax(l, -1) if scoring == "softmax" else torch.sigmoid(l)
    w = v.gather(-1, idx.long())
    return scale * (w / (w.sum(-1, keepdim=True) + (1e-20 if scoring == "sigmoid" else 0)) if renormalize else w)


def backward64(logits, idx, dw, scoring, renormalize, scale):
    """(dlogits, size of its terms); negative choices are none, one twice counts twice."""
    l = logits.double().detach().clone().requires_grad_()
    v = torch.softmax(l, -1) if scoring == "softmax" else torch.sigmoid(l)
    keep = (idx >= 0).double()
    w = v.gather(-1, idx.long().clamp(min=0)) * keep
    if renormalize and scoring == "softmax":  # the sum over all experts cancels: nothing of it is left, rounding included
        at = torch.where(idx >= 0, l.gather(-1, idx.long().clamp(min=0)), -torch.inf)
        at = torch.where(keep.sum(-1, keepdim=True) > 0, at, 0)
        w = torch.softmax(at, -1) * keep
    elif renormalize:
        total = w.sum(-1, keepdim=True) + (1e-20 if scoring == "sigmoid" else 0)
        w = torch.where(keep.sum(-1, keepdim=True) > 0, w / torch.where(total > 0, total, 1), 0)
    w = w * scale
    g = torch.where(idx >= 0, dw, 0).double()
    (w * g).sum().backward()
    with torch.no_grad():  # every term is at most w |g| and w sum |g| w
        w = w.abs()
        most = (w * g.abs()).sum(-1, keepdim=True)
        share = most * v / scale if scoring == "softmax" and not renormalize else 0
        at = (w * g.abs() + most * (w / abs(scale)))
        size = torch.zeros_like(l).scatter_add_(-1, idx.long().clamp(min=0), at * keep) + share
    return l.grad, size
