"""The norm's definition in 64 bits, for its tests."""
import torch

E4M3_MAX = 448.0


def rounded_sum(x, residual):
    """The sum as the stream holds it: one fp32 addition, rounded to the residual's type."""
    return x if residual is None else (x.float() + residual.float()).to(residual.dtype)


def norm64(h, weight, eps):
    h = h.double()
    rstd = (h.square().mean(-1) + eps) ** -0.5
    return h * rstd[..., None] * weight.double(), rstd


def scales64(y):
    """[..., ceil(C / 128)]: smallest power of two >= 2^-126 with max|y| <= 448 s; 1 for zeros.  Infinities and NaN count for none."""
    pad = torch.nn.functional.pad(torch.where(y.isfinite(), y.abs(), 0), (0, -y.shape[-1] % 128))
    top = pad.unflatten(-1, (-1, 128)).amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, m in [1/2, 1): 448 s = 0.875 2^(9 + k)
    k = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), k), 1.0)


def norm_backward64(dy, h, weight, rstd, dsum=None):
    """(dx, dweight, size of dx's terms, size of dweight's terms)."""
    dy, h, w, r = dy.double(), h.double(), weight.double(), rstd.double()[..., None]
    u, g = h * r, dy * w
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    size = r * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    if dsum is not None:
        dx, size = dx + dsum.double(), size + dsum.double().abs()
    rows = (dy * u).reshape(-1, h.shape[-1])
    return dx, rows.sum(0), size, rows.abs().sum(0)
