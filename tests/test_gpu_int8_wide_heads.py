"""The Q/K/V projection of many rows where its tiles of 256 channels x 256 rows do not fit the heads: an odd number of
heads of 128, so that the last tile is half empty and tiles lie across the ends of Q and K, with every part that the call
may leave out.  (By the estimate that chooses the kernel, each size here takes the one of 256 x 256 tiles by a third or more.)"""

import pytest
import torch

from hilberta_amd.flux_inputs import rotary_tables
from hilberta_amd.flux_int8 import Int8Rows, Int8Weight, int8_qkv, padded_features
from oracle import int8_ops as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _int8(gen, lead, features, scale):
    q = torch.zeros(*lead, padded_features(features), dtype=torch.int8, device="cuda")
    q[..., :features] = torch.randint(-127, 128, (*lead, features), generator=gen, device="cuda").to(torch.int8)
    return q, (torch.rand(*lead, generator=gen, device="cuda") + 0.5) * scale


def _set(gen, batch, rows, features, heads, dtype):
    columns = 3 * heads * 128
    randn = lambda n: torch.randn(n, generator=gen, device="cuda").to(dtype)  # noqa: E731
    return dict(x=Int8Rows(*_int8(gen, (batch, rows), features, 0.01), features, dtype),
                w=Int8Weight(*_int8(gen, (columns,), features, 0.01 * features**-0.5), features),
                bias=randn(columns), q=randn(128), k=randn(128))


def _call(sets, heads, **more):
    get = lambda name: [s[name] if s else None for s in sets]  # noqa: E731
    return int8_qkv(sets[0] and sets[0]["x"], sets[1]["x"], heads=heads, weights=get("w"), biases=get("bias"),
                    norms=(get("q"), get("k")), **more)


def _check(out, sets, heads, cos, sin, at=slice(None)):
    """The tokens ``at`` of every set of the out [3, B, T + n, heads, 128]."""
    first = 0
    for s in sets:
        if s is None:
            continue
        n = s["x"].q.shape[1]
        tokens = torch.arange(n, device="cuda")[at]
        p, d = O.linear(s["x"].q[:, tokens], s["x"].scale[:, tokens], s["w"].q, s["w"].scale, s["bias"])
        place = tokens + first
        norms = [None if s[k] is None else s[k].expand(len(tokens), -1) for k in "qk"]
        tables = (None, None) if cos is None else (cos[place], sin[place])
        for plane, (value, bound) in enumerate(O.qkv(p, d, heads, *norms, *tables)):
            O.held(out[plane][:, place], value, bound, "QKV"[plane])
        first += n


def _tables(T, n):
    at = torch.arange(n, device="cuda")
    ids = torch.zeros(T + n, 3, device="cuda")
    ids[T:, 1], ids[T:, 2] = at // 61, at % 61
    return rotary_tables(ids)


SIZES = [(2, 130, 3001, 11, 1102), (1, 33, 7777, 5, 1102), (2, 0, 5003, 9, 648), (3, 77, 2500, 7, 1400), (1, 0, 4099, 13, 1102),
         (2, 70, 4100, 13, 200)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,n,heads,features", SIZES)
def test_odd_heads(B, T, n, heads, features, dtype):
    gen = torch.Generator(device="cuda").manual_seed(n)
    sets = [_set(gen, B, rows, features, heads, dtype) if rows else None for rows in (T, n)]
    cos, sin = _tables(T, n)
    _check(_call(sets, heads, cos=cos, sin=sin), sets, heads, cos, sin)


@pytest.mark.parametrize("missing", ["rotation", "rotation and norms", "norms and biases", "rotation, norms and biases", "norm of K"])
@pytest.mark.parametrize("B,T,n,heads,features", SIZES[:3])
def test_parts_may_be_missing(B, T, n, heads, features, missing):
    gen = torch.Generator(device="cuda").manual_seed(n + 1)
    sets = [_set(gen, B, rows, features, heads, BF16) if rows else None for rows in (T, n)]
    for s in sets:
        if s:
            s.update(dict(q=None, k=None) if "norms" in missing else {}, **(dict(bias=None) if "biases" in missing else {}))
            s.update(dict(k=None) if "K" in missing else {})
    cos, sin = (None, None) if "rotation" in missing else _tables(T, n)
    _check(_call(sets, heads, cos=cos, sin=sin), sets, heads, cos, sin)


@pytest.mark.parametrize("B,T,n,heads,features", [SIZES[0], SIZES[4]])
def test_into_a_view_of_more_heads(B, T, n, heads, features):
    """What lies around the odd heads stays."""
    gen = torch.Generator(device="cuda").manual_seed(n + 2)
    sets = [_set(gen, B, rows, features, heads, BF16) if rows else None for rows in (T, n)]
    cos, sin = _tables(T, n)
    buf = torch.full((3, B, T + n + 3, heads + 1, 128), 5.0, dtype=BF16, device="cuda")
    view = buf[:, :, 1:1 + T + n, :heads]
    assert _call(sets, heads, cos=cos, sin=sin, out=view) is view
    _check(view, sets, heads, cos, sin, slice(None, None, 7))
    view.fill_(5.0)
    assert (buf == 5).all()
