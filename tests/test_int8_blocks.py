"""The plain form of the 8-bit blocks (oracle/int8_blocks.py) shows each mistake in their wiring: planted in it, every
one takes an output twice as far off as the blocks may be on the GPU (tests/int8_blocks.py)."""

import pytest
import torch

from oracle import int8_blocks as B
from oracle import int8_ops as O
from tests.int8_blocks import BOUND, off, raise_parameters

BF16 = torch.bfloat16
HEADS, T, N = 2, 13, 64
C, M = HEADS * 128, HEADS * 512


def _weight(gen, columns, features):
    q, scale, _ = O.quantize((torch.randn(columns, features, generator=gen) * features**-0.5).to(BF16))
    return q, scale, features


def _linear(gen, columns, features):
    return _weight(gen, columns, features), torch.zeros(columns, dtype=BF16)


def _tables():
    at = torch.arange(T + N, dtype=torch.float64)
    row, col = ((at - T).clamp(min=0) // 8, (at - T).clamp(min=0) % 8)
    angles = []
    for position, d in ((at * 0, 16), (row, 56), (col, 56)):
        angles.append(position[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    angles = torch.cat(angles, 1).repeat_interleave(2, 1)
    return angles.cos(), angles.sin()


def _mods(gen, count):
    return [0.7 * torch.randn(2, C, generator=gen) for _ in range(count)]


def _double():
    gen = torch.Generator().manual_seed(1)
    w = dict(qkv_x=_linear(gen, 3 * C, C), qkv_c=_linear(gen, 3 * C, C), out_x=_linear(gen, C, C), out_c=_linear(gen, C, C),
             ff_x=(_linear(gen, M, C), _linear(gen, C, M)), ff_c=(_linear(gen, M, C), _linear(gen, C, M)),
             **{n: torch.zeros(128, dtype=BF16) for n in ("norm_q", "norm_k", "norm_added_q", "norm_added_k")})
    raise_parameters(w, gen)
    cos, sin = _tables()
    x, c = torch.randn(2, N, C, generator=gen).to(BF16), torch.randn(2, T, C, generator=gen).to(BF16)
    mods = (_mods(gen, 6), _mods(gen, 6))
    xn, cn = (B.held8(O.adaln(r, m[0], m[1])[0]) for r, m in ((x, mods[0]), (c, mods[1])))
    return dict(w=w, mods=mods, x=x, xn=xn, c=c, cn=cn, cos=cos, sin=sin, next_mods=(_mods(gen, 2), _mods(gen, 2)), heads=HEADS)


def _single():
    gen = torch.Generator().manual_seed(2)
    w = dict(qkv=_linear(gen, 3 * C, C), mlp=_linear(gen, M, C), out=_linear(gen, C, C + M),
             **{n: torch.zeros(128, dtype=BF16) for n in ("norm_q", "norm_k")})
    raise_parameters(w, gen)
    cos, sin = _tables()
    h, mods = torch.randn(2, T + N, C, generator=gen).to(BF16), _mods(gen, 3)
    return dict(w=w, mods=mods, h=h, hn=B.held8(O.adaln(h, mods[0], mods[1])[0]), T=T, cos=cos, sin=sin, next_mods=_mods(gen, 2),
                heads=HEADS)


def _swap(*names):
    a, b = names
    return lambda s: s["w"].update({a: s["w"][b], b: s["w"][a]})


def _no_bias(name, at=None):
    def plant(s):
        old = s["w"][name]
        zero = lambda layer: (layer[0], torch.zeros_like(layer[1]))  # noqa: E731
        s["w"][name] = zero(old) if at is None else tuple(zero(x) if i == at else x for i, x in enumerate(old))
    return plant


def _planes(name, order):
    """Q, K and V of a projection in another order."""
    def plant(s):
        (q, scale, features), bias = s["w"][name]
        pick = torch.cat([torch.arange(C) + p * C for p in order])
        s["w"][name] = ((q[pick], scale[pick], features), bias[pick])
    return plant


def _ones(name):
    return lambda s: s["w"].update({name: torch.ones(128, dtype=BF16)})


def _mod(part, a, b):
    """Modulation vectors a and b of one row set exchanged."""
    def plant(s):
        m = list(s["mods"][part])
        m[a], m[b] = m[b], m[a]
        s["mods"] = tuple(m if i == part else x for i, x in enumerate(s["mods"]))
    return plant


def _exchange_out_columns(s):
    (q, scale, features), bias = s["w"]["out"]
    s["w"]["out"] = ((torch.cat([q[:, M:], q[:, :M]], 1), scale, features), bias)  # [mlp | attention]


ROTATION = {
    "no rotation": lambda s: s.update(cos=torch.ones_like(s["cos"]), sin=torch.zeros_like(s["sin"])),
    "rotation the other way": lambda s: s.update(sin=-s["sin"]),
    "rotation of the next token": lambda s: s.update(cos=s["cos"].roll(1, 0), sin=s["sin"].roll(1, 0)),
    "rotation of [image; text]": lambda s: s.update(cos=s["cos"].roll(-T, 0), sin=s["sin"].roll(-T, 0)),
    "no GELU": lambda s: s.update(act=lambda v: v),
    "no attention": lambda s: s.update(attend=lambda q, k, v: torch.zeros_like(v).flatten(2)),
    "a value's own row": lambda s: s.update(attend=lambda q, k, v: v.flatten(2)),
}

DOUBLE = {
    **ROTATION,
    **{f"{a} and {b} exchanged": _swap(a, b) for a, b in (("qkv_x", "qkv_c"), ("out_x", "out_c"), ("ff_x", "ff_c"), ("norm_q", "norm_k"),
                                                         ("norm_added_q", "norm_added_k"), ("norm_q", "norm_added_q"),
                                                         ("norm_k", "norm_added_k"))},
    **{f"no {n}": _ones(n) for n in ("norm_q", "norm_k", "norm_added_q", "norm_added_k")},
    **{f"no bias of {n}": _no_bias(n) for n in ("qkv_x", "qkv_c", "out_x", "out_c")},
    **{f"no bias of {n} {i}": _no_bias(n, i) for n in ("ff_x", "ff_c") for i in (0, 1)},
    **{f"{n} in order {o}": _planes(n, o) for n in ("qkv_x", "qkv_c") for o in ((1, 0, 2), (0, 2, 1), (2, 1, 0))},
    **{f"modulations {a} and {b} of set {p} exchanged": _mod(p, a, b) for p in (0, 1) for a, b in ((2, 5), (3, 4), (2, 3))},
    "the first modulation twice, image": lambda s: s.update(mods=((*s["mods"][0][:3], *s["mods"][0][:2], s["mods"][0][5]), s["mods"][1])),
    "the first modulation twice, text": lambda s: s.update(mods=(s["mods"][0], (*s["mods"][1][:3], *s["mods"][1][:2], s["mods"][1][5]))),
    "text and image modulations exchanged": lambda s: s.update(mods=s["mods"][::-1]),
    "text and image modulations that follow exchanged": lambda s: s.update(next_mods=s["next_mods"][::-1]),
    "shift and scale that follow exchanged": lambda s: s.update(next_mods=tuple(m[::-1] for m in s["next_mods"])),
}

SINGLE = {
    **ROTATION,
    "norm_q and norm_k exchanged": _swap("norm_q", "norm_k"),
    **{f"no {n}": _ones(n) for n in ("norm_q", "norm_k")},
    **{f"no bias of {n}": _no_bias(n) for n in ("qkv", "mlp", "out")},
    **{f"qkv in order {o}": _planes("qkv", o) for o in ((1, 0, 2), (0, 2, 1), (2, 1, 0))},
    "out over [mlp | attention]": _exchange_out_columns,
    "the scale as gate": lambda s: s.update(mods=(s["mods"][0], s["mods"][2], s["mods"][1])),
    "the shift as gate": lambda s: s.update(mods=(s["mods"][2], s["mods"][1], s["mods"][0])),
    "shift and scale that follow exchanged": lambda s: s.update(next_mods=s["next_mods"][::-1]),
}


def _copy(state):
    return {**state, "w": dict(state["w"])}


def _outputs(kind, state):
    """Q, K and V as attention is given them, the updates of the text and image rows, and the rows that follow."""
    given = []
    attend = state.get("attend", B.attend)
    state = {**state, "attend": lambda *heads: given.extend(heads) or attend(*heads)}
    if kind == "double":
        x, xn, c, cn = B.double_block(**state)
        return *given, x.double() - state["x"].double(), xn, c.double() - state["c"].double(), cn
    h, m = B.single_block(**state)
    update, t = h.double() - state["h"].double(), state["T"]
    return *given, update[:, :t], update[:, t:], B.held8(m)


@pytest.fixture(scope="module")
def right():
    states = dict(double=_double(), single=_single())
    return {k: (s, _outputs(k, s)) for k, s in states.items()}


@pytest.mark.parametrize("kind,mistake", [("double", m) for m in DOUBLE] + [("single", m) for m in SINGLE])
def test_each_mistake_shows(right, kind, mistake):
    state, want = right[kind]
    planted = _copy(state)
    (DOUBLE if kind == "double" else SINGLE)[mistake](planted)
    worst = max(off(a, b) for a, b in zip(_outputs(kind, planted), want))
    print(f"{kind}, {mistake}: {worst:.3f}")
    assert worst >= 2 * BOUND


def test_logits_are_as_the_bound_has_them(right):
    """Q and K around 1, so that logits are; rows' tops below 4.5 times their root mean square on average, and GELU's
    below 8 times."""
    state, _ = right["single"]
    seen = []
    B.single_block(**{**state, "attend": lambda q, k, v: seen.extend((q, k)) or B.attend(q, k, v),
                      "act": lambda v: seen.append(B.gelu(v)) or B.gelu(v)})
    rms = lambda t: t.double().square().mean(-1).sqrt()  # noqa: E731
    assert rms(seen[0]).mean() <= 1.2 and rms(seen[1]).mean() <= 1.2
    assert (seen[2].abs().amax(-1) / rms(seen[2])).mean() <= 8
    assert (state["hn"].abs().amax(-1) / rms(state["hn"])).mean() <= 4.5
