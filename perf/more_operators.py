"""16-bit linear layers with their epilogue and the image decoder's group norm: inputs, outputs and cost.

Two operators:

  linear  flux_linear.linear, residual + gate * act(x @ weight^T + bias) of 16-bit rows in one pass (act: none,
          GELU(tanh) or SiLU; bias, residual and gate where they are given), and flux_linear.linear_pair, the same
          of a text and an image row set, each by its own weight
  norm    flux_norm.group_norm, act(GroupNorm(x) * weight + bias) of images whose channels lie last in memory
          (act: none or SiLU), in 16 and 32 bits

Linear sizes are a 24-head, 3072-wide transformer's (the configuration of flux_model.FluxShape) at 1024 and
2048 px, a prompt's rows and one row, and generic odd ones.  Norm sizes are the stages of a decoder from latents of
1/8 resolution to 2048 px, 32 groups, and a generic odd one.  The drawn cases go over rows from one to the largest
image's, depths and widths that are no multiple of anything, rows that are part of a wider buffer, and maps of one
pixel to 2048 px in all types.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _linear(name, batch, rows, depth, columns, dtype="bf16", text=0, act="none", bias=True, residual=False, gate=False,
            part=False):
    return dict(kind="linear", name=name, batch=batch, text=text, rows=rows, depth=depth, columns=columns, dtype=dtype,
                act=act, bias=bias, residual=residual, gate=gate, part=part)


def _norm(name, batch, height, width, channels, groups, dtype="bf16", act="silu"):
    return dict(kind="norm", name=name, batch=batch, height=height, width=width, channels=channels, groups=groups,
                dtype=dtype, act=act)


def listed():
    return [
        # a modulation of one row: the read of the weights, and the launch
        _linear("linear one row", 1, 1, 3072, 18432),
        # the text states of a short prompt, in the other 16-bit type
        _linear("linear 77 rows", 1, 77, 4096, 3072, dtype="fp16"),
        # nothing a multiple of anything, a plain residual, rows that are part of a wider buffer
        _linear("linear odd", 3, 333, 1001, 777, dtype="fp16", act="silu", bias=False, residual=True, part=True),
        # the text rows' way out of their MLP into the residual stream: few rows, a long sum
        _linear("linear 512 rows gated", 1, 512, 12288, 3072, residual=True, gate=True),
        # the joint Q/K/V projection of a double block at 1024 px: two row sets, two weights
        _linear("linear pair 1024px", 1, 4096, 3072, 9216, text=512),
        # two 1024 px images into the MLP
        _linear("linear 1024px b2 gelu", 2, 4096, 3072, 12288, act="gelu"),
        # the image rows' way out of their MLP into the residual stream at 2048 px
        _linear("linear 2048px gated", 1, 16384, 12288, 3072, residual=True, gate=True),
        # a thumbnail's deepest stage: the launches
        _norm("norm 16x16", 1, 16, 16, 512, 32),
        # five channels a group, nothing a multiple of anything, no activation
        _norm("norm odd", 3, 37, 53, 60, 12, dtype="fp16", act="none"),
        # the deepest stage of a 1024 px image
        _norm("norm 128x128", 1, 128, 128, 512, 32),
        # a middle stage of a 1024 px image in 32 bits
        _norm("norm 512x512 fp32", 1, 512, 512, 256, 32, dtype="fp32"),
        # the last stage of a 2048 px image
        _norm("norm 2048x2048", 1, 2048, 2048, 128, 32),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST = 16384 * 12288 * 3072  # products of the largest listed linear case
MOST_VALUES = 2048 * 2048 * 128  # values of the largest listed norm case


def draw(rng):
    batch = rng.choice((1, 1, 1, 2, 3))
    if rng.random() < 0.6:
        rows, depth, columns = _log(rng, 1, 16384), _log(rng, 8, 15360), _log(rng, 8, 18432)
        if rng.random() < 0.5:  # (a model's widths)
            depth, columns = -(-depth // 64) * 64, -(-columns // 64) * 64
        text = rng.choice((0, 0, 0, _log(rng, 1, 700), 512))
        rows = max(1, min(rows, MOST // (batch * depth * columns) - text))
        residual = rng.random() < 0.5
        return dict(kind="linear", batch=batch, text=text, rows=rows, depth=depth, columns=columns,
                    dtype=rng.choice(("bf16", "bf16", "fp16")), act=rng.choice(("none", "none", "gelu", "silu")),
                    bias=rng.random() < 0.8, residual=residual, gate=residual and rng.random() < 0.5,
                    part=rng.random() < 0.2)
    groups = rng.choice((32, 32, 32, 16, 8, _log(rng, 1, 64)))
    channels = groups * rng.choice((1, 2, 4, 8, 16, 3, 5, 10, 20))
    height = _log(rng, 1, 2048)
    width = min(2048, max(1, round(height * rng.uniform(0.5, 2))))
    height = max(1, min(height, MOST_VALUES // (batch * width * channels)))
    return dict(kind="norm", batch=batch, height=height, width=width, channels=channels, groups=groups,
                dtype=rng.choice(("bf16", "fp16", "fp32")), act=rng.choice(("silu", "silu", "none")))


# ------------------------------------------------------------------ inputs
def _rows(gen, shape, dtype, part=False):
    """Activations: N(0, 1) with one channel in 64 some eight times as large, as transformers have them; with `part`
    as a column block of a buffer 64 values wider."""
    x = torch.randn(*shape[:-1], shape[-1] + 64 * part, generator=gen, device="cuda")
    loud = torch.rand(x.shape[-1], generator=gen, device="cuda") < 1 / 64
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)[..., :shape[-1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, batch = DTYPES[case["dtype"]], case["batch"]

    def normal(*shape, mean=0.0, std=1.0):
        return (mean + std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

    if case["kind"] == "linear":
        depth, columns, sets = case["depth"], case["columns"], []
        for rows in (case["text"], case["rows"]):
            if not rows:
                continue
            sets.append(dict(
                x=_rows(gen, (batch, rows, depth), dtype, case["part"]),
                weight=normal(columns, depth, std=depth**-0.5),
                bias=normal(columns, std=0.02) if case["bias"] else None,
                residual=_rows(gen, (batch, rows, columns), dtype) if case["residual"] else None,
                gate=normal(batch, columns, std=0.2) if case["gate"] else None))
        return dict(case=case, sets=sets)
    channels = case["channels"]
    # maps whose channels have means and sizes of their own
    x = torch.randn(batch, case["height"], case["width"], channels, generator=gen, device="cuda")
    x *= 0.5 + torch.rand(channels, generator=gen, device="cuda")
    x += 2 * torch.randn(channels, generator=gen, device="cuda")
    return dict(case=case, x=x.to(dtype).permute(0, 3, 1, 2), weight=normal(channels, mean=1.0, std=0.1),
                bias=normal(channels, std=0.1))


# ------------------------------------------------------------------ the plain forms
def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v / (1 + torch.exp(-v)) if act == "silu" else v


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "linear":
        done = []
        for s in state["sets"]:
            out = torch.matmul(s["x"].float(), s["weight"].float().t())
            if s["bias"] is not None:
                out = out + s["bias"].float()
            out = _act(out, case["act"])
            if s["gate"] is not None:
                out = out * s["gate"].float()[:, None]
            if s["residual"] is not None:
                out = s["residual"].float() + out
            done.append(out.to(dtype))
        return tuple(done)
    x = state["x"].float()
    g = x.unflatten(1, (case["groups"], -1))
    mean = g.mean((2, 3, 4), keepdim=True)
    d = g - mean
    n = d * torch.rsqrt((d * d).mean((2, 3, 4), keepdim=True) + EPS)
    y = n.flatten(1, 2) * state["weight"].float()[:, None, None] + state["bias"].float()[:, None, None]
    return _act(y, case["act"]).to(dtype).contiguous(memory_format=torch.channels_last)


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    case = state["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["kind"] == "linear":
        from hilberta_amd.flux_linear import linear, linear_pair

        if len(state["sets"]) == 2:
            return linear_pair(*state["sets"], act=act)
        s = state["sets"][0]
        return (linear(s["x"], s["weight"], s["bias"], act=act, residual=s["residual"], gate=s["gate"]),)
    from hilberta_amd.flux_norm import group_norm

    return group_norm(state["x"], case["groups"], state["weight"], state["bias"], act=act, eps=EPS)


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------ what they cannot do without
def work(case):
    if case["kind"] == "linear":
        B, K, N = case["batch"], case["depth"], case["columns"]
        M, sets = B * (case["rows"] + case["text"]), 1 + (case["text"] > 0)
        weights = sets * N * (K + case["bias"] + B * case["gate"])
        return dict(bytes=2 * (M * K + weights + M * N * (1 + case["residual"])), flops=2 * M * K * N)
    values = case["batch"] * case["height"] * case["width"] * case["channels"]
    # two sums, the difference, the product with the weight and the bias; an exponential and a quotient
    return dict(bytes=(2 * values + 2 * case["channels"]) * DTYPES[case["dtype"]].itemsize,
                flops=values * (6 + 4 * (case["act"] == "silu")))


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f8 = lambda t: t.to(torch.float64)  # noqa: E731
    act = {"none": lambda v: v, "silu": lambda v: v * torch.special.expit(v),
           "gelu": lambda v: v * torch.special.expit(math.sqrt(8 / math.pi) * (v + 0.044715 * v**3))}[case["act"]]
    if case["kind"] == "linear":
        done = []
        for a in s["sets"]:
            x, w = f8(a["x"]).flatten(0, 1), f8(a["weight"])
            out = torch.mm(x, w.T) if a["bias"] is None else torch.addmm(f8(a["bias"]), x, w.T)
            out = act(out.view(*a["x"].shape[:2], -1))
            if a["residual"] is not None:
                scale = torch.ones_like(out[:, :1]) if a["gate"] is None else f8(a["gate"]).unsqueeze(1)
                out = torch.addcmul(f8(a["residual"]), out, scale)
            done.append(out)
        return tuple(done)
    x = f8(s["x"])
    B, C = x.shape[:2]
    per = C // case["groups"]
    # each channel's mean and mean square, then its group's
    flat = x.permute(0, 2, 3, 1).reshape(B, -1, C)
    var, mean = torch.var_mean(flat, dim=1, correction=0)
    group = mean.view(B, -1, per)
    center = group.mean(2, keepdim=True)
    spread = (var.view(B, -1, per) + (group - center).square()).mean(2, keepdim=True)
    center, spread = (t.expand(-1, -1, per).reshape(B, 1, C) for t in (center, spread))
    y = (flat - center) / (spread + EPS).sqrt() * f8(s["weight"]) + f8(s["bias"])
    return act(y).view(B, *x.shape[2:], C).permute(0, 3, 1, 2)
