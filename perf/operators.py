"""The denoiser's 8-bit linear layers: what they take, what they return and what they cost.

Three operators, each as the transformer's blocks call it:

  linear   int8_linear of 16-bit rows: the rows to 8 bits by their own scale, the product with a weight
           of one scale a channel, bias, GELU(tanh) where it is asked for
  adaln    adaln_quantize and int8_linear: gated residual, LayerNorm and modulation straight into 8-bit
           rows, and the product that reads them (the way into an MLP)
  qkv      int8_qkv of 8-bit rows: the text and image rows' Q/K/V projections with the heads' RMSNorm of
           Q and K and the position rotation, written as the joint [text; image] heads of attention

Sizes are a 24-head, 3072-wide transformer's (the configuration of flux_model.FluxShape) at 1024 and
2048 px, its single rows, and generic odd ones.  The drawn cases go over rows from one to the largest
image's, both 16-bit types, odd depths, widths, head counts and batches.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEAD_DIM = 128
EPS = 1e-6
AXES_DIM, THETA = (16, 56, 56), 10000.0


def _linear(name, batch, rows, depth, columns, dtype="bf16", bias=True, gelu=False):
    return dict(kind="linear", name=name, batch=batch, rows=rows, depth=depth, columns=columns, dtype=dtype,
                bias=bias, gelu=gelu)


def _adaln(name, batch, rows, hidden, columns, dtype="bf16", residual=True):
    return dict(kind="adaln", name=name, batch=batch, rows=rows, hidden=hidden, columns=columns, dtype=dtype,
                residual=residual)


def _qkv(name, batch, text, image, heads, depth, dtype="bf16"):
    return dict(kind="qkv", name=name, batch=batch, text=text, image=image, heads=heads, depth=depth, dtype=dtype)


def listed():
    return [
        # a modulation of one row: the read of the weights, and the launches
        _linear("linear one row", 1, 1, 3072, 18432),
        # the text states of a short prompt, in the other 16-bit type
        _linear("linear 77 rows", 1, 77, 4096, 3072, dtype="fp16"),
        # nothing a multiple of anything
        _linear("linear odd", 2, 333, 1000, 777, dtype="fp16", bias=False, gelu=True),
        # the text rows' way out of their MLP: few rows, a long sum
        _linear("linear 512 rows", 1, 512, 12288, 3072),
        # the image rows' way out of their MLP at 2048 px
        _linear("linear 2048px", 1, 16384, 12288, 3072),
        # a short model's rows, with no residual yet (the first block)
        _adaln("adaln 64 rows", 1, 64, 512, 2048, dtype="fp16", residual=False),
        # two 1024 px images into the MLP
        _adaln("adaln 1024px b2", 2, 4096, 3072, 12288),
        # the joint rows of a single block at 2048 px
        _adaln("adaln 2048px", 1, 16896, 3072, 12288),
        # one token
        _qkv("qkv one row", 1, 0, 1, 24, 3072),
        # an odd head count, odd rows on both sides, a batch
        _qkv("qkv odd", 3, 77, 451, 5, 648, dtype="fp16"),
        # a double block at 1024 px
        _qkv("qkv 1024px", 1, 512, 4096, 24, 3072),
        # a double block at 2048 px
        _qkv("qkv 2048px", 1, 512, 16384, 24, 3072),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST = 16384 * 12288 * 3072  # products of the largest listed case


def draw(rng):
    kind = rng.choice(("linear", "adaln", "qkv"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    batch = rng.choice((1, 1, 1, 2, 3))
    rows = _log(rng, 1, 16384)
    if kind == "linear":
        depth, columns = _log(rng, 48, 15360), _log(rng, 16, 18432)
        rows = max(1, min(rows, MOST // (batch * depth * columns)))
        return dict(kind=kind, batch=batch, rows=rows, depth=depth, columns=columns, dtype=dtype,
                    bias=rng.random() < 0.7, gelu=rng.random() < 0.3)
    if kind == "adaln":
        hidden, columns = 8 * _log(rng, 16, 512), _log(rng, 64, 14000)
        rows = max(1, min(rows, MOST // (batch * hidden * columns)))
        return dict(kind=kind, batch=batch, rows=rows, hidden=hidden, columns=columns, dtype=dtype,
                    residual=rng.random() < 0.8)
    heads, depth = _log(rng, 1, 32), _log(rng, 64, 4200)
    text = rng.choice((0, 1, _log(rng, 1, 700), 512))
    rows = max(1, min(rows, MOST // (batch * depth * heads * 3 * HEAD_DIM) - text))
    return dict(kind=kind, batch=batch, text=text, image=rows, heads=heads, depth=depth, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _rows(gen, shape, dtype):
    """Activations: N(0, 1) with one channel in 64 some eight times as large, as transformers have them."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 1 / 64
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _eight_bits(x, depth):
    """x [..., depth] as whole numbers by each row's largest value, rows filled up with zeros to a multiple
    of 64, and the scales."""
    scale = x.abs().amax(-1) / 127
    q = torch.zeros(*x.shape[:-1], -(-depth // 64) * 64, dtype=torch.int8, device=x.device)
    q[..., :depth] = torch.round(x / scale.clamp_min(1e-30)[..., None]).to(torch.int8)
    return q, scale


def _weight(gen, columns, depth):
    """An 8-bit weight [columns, depth] of N(0, 1 / depth) and its channels' scales."""
    return _eight_bits(torch.randn(columns, depth, generator=gen, device="cuda") * depth**-0.5, depth)


def _vector(gen, n, dtype, mean=0.0, std=0.02):
    return (mean + std * torch.randn(n, generator=gen, device="cuda")).to(dtype)


def _rotary(text, image):
    """cos and sin rows of text ids (0, 0, 0) and image ids (0, row, column) of a square-ish raster."""
    side = max(1, math.isqrt(image))
    at = torch.arange(image, device="cuda")
    ids = torch.zeros(text + image, 3, dtype=torch.float64, device="cuda")
    ids[text:, 1], ids[text:, 2] = at // side, at % side
    angles = torch.cat([ids[:, a:a + 1] * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
                        for a, d in enumerate(AXES_DIM)], 1).repeat_interleave(2, 1)
    return angles.cos().float(), angles.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, batch = DTYPES[case["dtype"]], case["batch"]
    state = dict(case=case)
    if case["kind"] == "linear":
        state["x"] = _rows(gen, (batch, case["rows"], case["depth"]), dtype)
        state["w"], state["ws"] = _weight(gen, case["columns"], case["depth"])
        state["bias"] = _vector(gen, case["columns"], dtype) if case["bias"] else None
    elif case["kind"] == "adaln":
        hidden, columns = case["hidden"], case["columns"]
        state["x"] = _rows(gen, (batch, case["rows"], hidden), dtype)
        mod = (torch.randn(batch, 3 * hidden, generator=gen, device="cuda") * 0.2).to(dtype)
        state["shift"], state["scale"], state["gate"] = mod.chunk(3, 1)
        state["y"] = _rows(gen, (batch, case["rows"], hidden), dtype) if case["residual"] else None
        state["x_out"] = torch.empty_like(state["x"]) if case["residual"] else None
        state["w"], state["ws"] = _weight(gen, columns, hidden)
        state["bias"] = _vector(gen, columns, dtype)
    else:
        depth, columns = case["depth"], 3 * case["heads"] * HEAD_DIM
        for part in ("text", "image"):
            state[part] = None
            if case[part]:
                q, s = _eight_bits(_rows(gen, (batch, case[part], depth), dtype).float(), depth)
                w, ws = _weight(gen, columns, depth)
                state[part] = dict(q=q, s=s, w=w, ws=ws, bias=_vector(gen, columns, dtype),
                                   norm_q=_vector(gen, HEAD_DIM, dtype, 1.0, 0.1),
                                   norm_k=_vector(gen, HEAD_DIM, dtype, 1.0, 0.1))
        state["cos"], state["sin"] = _rotary(case["text"], case["image"])
    return state


# ------------------------------------------------------------------ the plain forms
def _product(q, s, w, ws, bias):
    """fp32 rows of the product of 8-bit rows (values and their scales) with an 8-bit weight."""
    out = torch.matmul(q.float(), w.float().t()) * s[..., None] * ws
    return out if bias is None else out + bias.float()


def _gelu(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _to_eight_bits(x):
    """Rows of fp32 values as whole numbers in [-127, 127] (still fp32) and scales."""
    top = x.abs().amax(-1)
    return torch.round(x * 127 / torch.where(top > 0, top, 1.0)[..., None]), top / 127


def _plain(state):
    case = state["case"]
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    if kind == "linear":
        q, s = _to_eight_bits(state["x"].float())
        out = _product(q, s, state["w"][:, :case["depth"]], state["ws"], state["bias"])
        return (_gelu(out) if case["gelu"] else out).to(dtype)
    if kind == "adaln":
        r = state["x"].float()
        if case["residual"]:
            r = r + state["gate"].float()[:, None] * state["y"].float()
        d = r - r.mean(-1, keepdim=True)
        n = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
        q, s = _to_eight_bits(state["shift"].float()[:, None] + n * (1 + state["scale"].float()[:, None]))
        out = _gelu(_product(q, s, state["w"][:, :case["hidden"]], state["ws"], state["bias"])).to(dtype)
        return (out, r.to(dtype)) if case["residual"] else (out,)
    parts = [state[part] for part in ("text", "image") if state[part]]
    p = torch.cat([_product(a["q"], a["s"], a["w"], a["ws"], a["bias"]) for a in parts], 1)
    p = p.unflatten(-1, (3, case["heads"], HEAD_DIM))
    qk, v = p[:, :, :2], p[:, :, 2]
    w = torch.cat([torch.stack([a["norm_q"], a["norm_k"]]).float()[None].expand(a["q"].shape[1], -1, -1)
                   for a in parts])[:, :, None]
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    even, odd = qk[..., 0::2], qk[..., 1::2]
    cos, sin = state["cos"][:, None, None], state["sin"][:, None, None]
    qk = torch.stack([even * cos[..., 0::2] - odd * sin[..., 0::2],
                      odd * cos[..., 1::2] + even * sin[..., 1::2]], -1).flatten(-2)
    return qk[:, :, 0].to(dtype), qk[:, :, 1].to(dtype), v.to(dtype)


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    from hilberta_amd.flux_int8 import Int8Rows, Int8Weight, adaln_quantize, int8_linear, int8_qkv

    case = state["case"]
    kind = case["kind"]
    if kind == "linear":
        weight = Int8Weight(state["w"], state["ws"], case["depth"])
        return int8_linear(state["x"], weight, state["bias"], gelu=case["gelu"])
    if kind == "adaln":
        rows = adaln_quantize(state["x"], state["shift"], state["scale"], y=state["y"],
                              gate=state["gate"] if case["residual"] else None, x_out=state["x_out"], eps=EPS)
        out = int8_linear(rows, Int8Weight(state["w"], state["ws"], case["hidden"]), state["bias"], gelu=True)
        return (out, state["x_out"]) if case["residual"] else (out,)
    dtype, depth = DTYPES[case["dtype"]], case["depth"]
    t, i = state["text"], state["image"]
    out = int8_qkv(
        t and Int8Rows(t["q"], t["s"], depth, dtype), Int8Rows(i["q"], i["s"], depth, dtype), heads=case["heads"],
        weights=(t and Int8Weight(t["w"], t["ws"], depth), Int8Weight(i["w"], i["ws"], depth)),
        biases=(t and t["bias"], i["bias"]),
        norms=((t and t["norm_q"], i["norm_q"]), (t and t["norm_k"], i["norm_k"])),
        eps=EPS, cos=state["cos"], sin=state["sin"])
    return out[0], out[1], out[2]


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------ what they cannot do without
def work(case):
    kind, B = case["kind"], case["batch"]
    if kind == "linear":
        M, K, N = B * case["rows"], case["depth"], case["columns"]
        return dict(bytes=2 * M * K + N * (K + 4) + 2 * N * case["bias"] + 2 * M * N, flops=2 * M * K * N)
    if kind == "adaln":
        M, K, N = B * case["rows"], case["hidden"], case["columns"]
        # x (y and the gate) in, the residual out; the 8-bit rows stay inside
        rows = 2 * M * K * (3 if case["residual"] else 1) + 2 * B * K * (3 if case["residual"] else 2)
        return dict(bytes=rows + N * (K + 6) + 2 * M * N, flops=2 * M * K * N)
    K, N, tokens = case["depth"], 3 * case["heads"] * HEAD_DIM, case["text"] + case["image"]
    weights = (1 + (case["text"] > 0)) * N * (K + 6)
    return dict(bytes=B * tokens * (K + 4) + weights + 8 * tokens * HEAD_DIM + 2 * B * tokens * N,
                flops=2 * B * tokens * K * N)


# ------------------------------------------------------------------ the definition, in 64 bits
def _rounded(x):
    """The operators' 8-bit rows of 64-bit values: (whole numbers, scale [..., 1])."""
    top = x.abs().max(dim=-1, keepdim=True).values
    return (x * 127 / top).round(), top / 127


def exact(case, seed):
    s = prepare(case, seed)
    f8 = lambda t: t.to(torch.float64)  # noqa: E731
    gelu = lambda v: v * torch.special.expit(math.sqrt(8 / math.pi) * (v + 0.044715 * v**3))  # noqa: E731
    if case["kind"] == "linear":
        q, scale = _rounded(f8(s["x"]))
        out = torch.mm(q.flatten(0, 1), f8(s["w"][:, :case["depth"]]).T).view(*s["x"].shape[:2], -1)
        out = out * scale * f8(s["ws"])
        if s["bias"] is not None:
            out = out + f8(s["bias"])
        return gelu(out) if case["gelu"] else out
    if case["kind"] == "adaln":
        r = f8(s["x"])
        if s["y"] is not None:
            r = torch.addcmul(r, f8(s["gate"]).unsqueeze(1), f8(s["y"]))
        var, mean = torch.var_mean(r, dim=-1, correction=0, keepdim=True)
        m = (r - mean) / (var + EPS).sqrt() * (f8(s["scale"]).unsqueeze(1) + 1) + f8(s["shift"]).unsqueeze(1)
        q, scale = _rounded(m)
        out = torch.mm(q.flatten(0, 1), f8(s["w"][:, :case["hidden"]]).T).view(*r.shape[:2], -1)
        out = gelu(out * scale * f8(s["ws"]) + f8(s["bias"]))
        return (out, r) if s["y"] is not None else (out,)
    heads, done = case["heads"], []
    turn = torch.complex(f8(s["cos"][:, 0::2]), f8(s["sin"][:, 0::2]))
    first = 0
    for part in ("text", "image"):
        a = s[part]
        if a is None:
            continue
        n = a["q"].shape[1]
        p = torch.mm(f8(a["q"]).flatten(0, 1), f8(a["w"]).T) * f8(a["s"]).view(-1, 1) * f8(a["ws"]) + f8(a["bias"])
        q, k, v = p.view(-1, n, 3, heads, HEAD_DIM).unbind(2)
        made = []
        for x, w in ((q, a["norm_q"]), (k, a["norm_k"])):
            x = x / (x.pow(2).sum(-1, keepdim=True) / HEAD_DIM + EPS).sqrt() * f8(w)
            x = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn[first:first + n, None]
            made.append(torch.view_as_real(x).flatten(-2))
        done.append((*made, v))
        first += n
    return tuple(torch.cat(x, 1) for x in zip(*done))
