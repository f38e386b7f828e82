"""The 16-bit linear layers of hilberta_amd.flux_linear and the group norm of hilberta_amd.flux_norm in 64 bits, and
how far fp32 may be from them.

Each function returns values and a bound on a kernel's error before the last rounding; ``held`` adds that rounding.
A rounding is off by half a step: eps / 2 of the value.
"""

import math

import torch

U = 2.0**-24  # half a step of fp32


def activate(v, act):
    if act == "gelu":
        return v * torch.special.expit(math.sqrt(8 / math.pi) * (v + 0.044715 * v**3))
    return v * torch.special.expit(v) if act == "silu" else v


def linear(x, weight, bias=None, act=None, residual=None, gate=None):
    """(out, bound) of residual + gate * act(x @ weight^T + bias), x [B, rows, K] or [rows, K].

    Products of 16-bit values are exact in fp32 (22 bits); each of the K additions and the bias is off by U of what has
    been added, at most the sum of magnitudes.  GELU and SiLU have slopes up to 1.13; the exponential of an argument e,
    itself off by 3 U, changes v s (s = 1 / (1 + exp e)) by |v| s (1 - s) |e| 3 U <= 0.28 |v| 3 U, and exponential,
    sum, reciprocal and product add at most 8 U of |v|.  Gate and residual are two more roundings."""
    x, w = x.double(), weight.double()
    p, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        p, size = p + bias.double(), size + bias.double().abs()
    bound = (x.shape[-1] + 2) * U * size
    out = activate(p, act)
    if act is not None:
        bound = 1.13 * bound + 9 * U * p.abs()
    if residual is not None:
        g = 1.0 if gate is None else gate.double().unsqueeze(1) if x.ndim == 3 else gate.double()
        out, bound = out * g, bound * abs(g)
        bound = bound + 2 * U * (out.abs() + residual.double().abs())
        out = out + residual.double()
    return out, bound


def held(got, exact, bound):
    """Whether ``got`` is ``exact`` rounded once to its type, given a value before the rounding within ``bound``."""
    info = torch.finfo(got.dtype)
    step = torch.maximum(exact.abs() + bound, torch.tensor(info.smallest_normal, dtype=torch.float64, device=exact.device))
    return (got.double() - exact).abs() <= bound + info.eps / 2 * step


def relative(got, exact):
    return ((got.double() - exact).norm() / exact.norm().clamp_min(1e-30)).item()


def group_norm(x, groups, weight=None, bias=None, act=None, eps=1e-6, steps=99, statistics=None):
    """(out, bound) of act(GroupNorm(x) * weight + bias), x [B, pixels, C].

    A kernel's mean comes of ``steps`` additions and joins, each off by U of at most the mean's size plus the deviation:
    16 joins of a thread's pixels, 67 additions over the workgroup's threads and 16 joins of chunks where nothing else is
    said.  Its variance's relative error is twice that count of U and the square of the mean's error in deviations, halved
    by the root.  Then come the difference, the two products, the sum, and SiLU as in ``linear``.  ``statistics``: mean
    and variance [B, 1, groups, 1], where x is a part of the image."""
    B, P, C = x.shape
    v = x.double().reshape(B, P, groups, C // groups)
    mean, var = statistics or (v.mean((1, 3), keepdim=True), v.var((1, 3), keepdim=True, unbiased=False))
    std = (var + eps).sqrt()
    dmean = steps * U * (mean.abs() + var.sqrt())
    n = (v - mean) / std
    dn = (dmean + U * (v - mean).abs()) / std + n.abs() * (steps * U + (dmean / std) ** 2 + 4 * U)
    n, dn = n.reshape(B, P, C), dn.reshape(B, P, C)
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    y = n * w + b
    bound = dn * abs(w) + 2 * U * ((n * w).abs() + abs(b))
    if act == "silu":
        bound = 1.13 * bound + 9 * U * y.abs()
    return activate(y, act), bound
