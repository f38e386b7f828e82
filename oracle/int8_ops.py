"""The 8-bit linear layers of hilberta_amd.flux_int8 in 64 bits, and how far fp32 may be from them.

Each function returns values and, where a kernel computes in fp32, a bound on its error before the last
rounding; ``held`` adds that rounding.  A rounding is off by half a step: eps / 2 of the value.
"""

import math

import torch

U = 2.0**-24  # half a step of fp32


def quantize(x):
    """(q int64, scale float64, quotient float64) of rows x [..., K]: exact, ties to even."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    y = torch.where(top > 0, 127 * x / torch.where(top > 0, top, 1.0), 0.0)
    return torch.round(y).long(), (top / 127)[..., 0], y


def adaln(x, shift, scale, y=None, gate=None, eps=1e-6):
    """(m, bound of m's error, r, bound of r's error) for m = shift + LayerNorm(r) (1 + scale)."""
    x, sh, sc = x.double(), shift.double()[:, None], scale.double()[:, None]
    r, dr = x, torch.zeros_like(x)
    if y is not None:
        gy = gate.double()[:, None] * y.double()
        r = x + gy
        dr = 2 * U * (x.abs() + gy.abs())
    hidden = r.shape[-1]
    mean, var = r.mean(-1, keepdim=True), r.var(-1, keepdim=True, unbiased=False)
    rstd = (var + eps).rsqrt()
    n = (r - mean) * rstd
    # a lane adds 8 ceil(hidden / 512) values (8 at a time in rows the kernel rounds up to 16 vectors), six
    # exchanges follow: each addition off by U of what has been added
    adds = 8 * 16 + 6
    dmean = adds * U * r.abs().mean(-1, keepdim=True) + dr.mean(-1, keepdim=True)
    dd = dr + dmean + U * (r - mean).abs()
    # relative: of the sum of squares (additions, squares, and the differences' own errors), halved by the root
    dvar = (adds + 2) * U + 2 * (dd * (r - mean).abs()).mean(-1, keepdim=True) / (var + eps)
    dn = dd * rstd + n.abs() * (dvar / 2 + 3 * U)
    m = sh + n * (1 + sc)
    return m, dn * (1 + sc).abs() + 3 * U * (n * (1 + sc)).abs() + U * m.abs(), r, dr


def linear(q, scale, w, w_scale, bias=None, features=None):
    """(p, bound of its error) for 8-bit rows q [..., K'] and weight w [N, K']."""
    acc = (q.double().flatten(0, -2) @ w.double().t()).unflatten(0, q.shape[:-1])
    v = acc * scale.double()[..., None] * w_scale.double()
    # the sum to fp32, two products; then the bias and its sum
    p, d = v, 3 * U * v.abs()
    if bias is not None:
        p = v + bias.double()
        d = d + U * (v.abs() + bias.double().abs())
    return p, d


def gelu(p, d):
    """GELU(tanh) of values p off by d."""
    u = math.sqrt(2 / math.pi) * (p + 0.044715 * p**3)
    g = p * torch.sigmoid(2 * u)
    # exp2 of an argument off by 4 U of itself; where that is past 60 the value is below 1e-17 of p
    return g, 1.13 * d + g.abs() * 2.0**-16 + 1e-17 * p.abs()


def qkv(p, d, heads, norm_q, norm_k, cos, sin, eps=1e-6):
    """[Q, K, V] each (value, bound) [B, N, heads, 128] of projections p, d [B, N, 3 heads 128]; norms are
    [N, 128] rows or None."""
    p, d = p.unflatten(-1, (3, heads, 128)), d.unflatten(-1, (3, heads, 128))
    out = []
    for plane, norm in ((0, norm_q), (1, norm_k)):
        x, dx = p[:, :, plane], d[:, :, plane]
        ms = x.square().mean(-1, keepdim=True)
        r = (ms + eps).rsqrt()
        w = torch.ones(128, dtype=torch.float64, device=x.device) if norm is None else norm.double()[:, None]
        n = x * r * w
        # the mean of squares: 130 roundings at most, and the values' own errors
        dms = 132 * U + 2 * (dx * x.abs()).mean(-1, keepdim=True) / (ms + eps)
        dn = dx * r * w.abs() + n.abs() * (dms / 2 + 4 * U)
        if cos is not None:
            c, s = cos.double()[:, None], sin.double()[:, None]
            turned = torch.stack([-n[..., 1::2], n[..., 0::2]], -1).flatten(-2)
            dturned = torch.stack([dn[..., 1::2], dn[..., 0::2]], -1).flatten(-2)
            dn = dn * c.abs() + dturned * s.abs() + 3 * U * ((n * c).abs() + (turned * s).abs())
            n = n * c + turned * s
        out.append((n, dn))
    return [*out, (p[:, :, 2], d[:, :, 2])]


def held(got, value, bound, what=""):
    """Assert that 16-bit ``got`` is ``value`` off by ``bound`` and one rounding."""
    info = torch.finfo(got.dtype)
    off = (got.double() - value).abs()
    allowed = bound + info.eps / 2 * (value.abs() + bound) + info.smallest_normal * info.eps / 2
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off / allowed).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the allowed error"
    return worst
