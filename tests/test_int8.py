"""The 8-bit linear layers' refusals and their 64-bit oracle, on the CPU.

The operators make their checks on any device and refuse CPU tensors last, so every refusal is seen here
without a GPU; the C entry points return HB_EINVAL before any HIP call.
"""

import ctypes
import math

import pytest
import torch

from hilberta_amd import _lib
from hilberta_amd import flux_int8 as f
from oracle import int8_ops as O

BF16, FP16 = torch.bfloat16, torch.float16
ON_DEVICE = "device tensors"


def _rows(*lead, features=70, dtype=BF16):
    return f.Int8Rows(torch.zeros(*lead, f.padded_features(features), dtype=torch.int8), torch.zeros(lead), features, dtype)


def _weight(columns, features=70):
    return f.Int8Weight(torch.zeros(columns, f.padded_features(features), dtype=torch.int8), torch.zeros(columns), features)


def _refused(match, call, *args, **kwargs):
    with pytest.raises(ValueError, match=match):
        call(*args, **kwargs)


# ------------------------------------------------------------------ entry points
def test_padded_features():
    assert [f.padded_features(n) for n in (1, 63, 64, 65, 12288)] == [64, 64, 64, 128, 12288]


def test_quantize_refusals():
    q = f.quantize_rows
    _refused(ON_DEVICE, q, torch.zeros(3, 5, dtype=BF16))
    _refused(ON_DEVICE, q, torch.zeros(2, 0, 5, dtype=FP16))
    _refused("bf16 or fp16", q, torch.zeros(3, 5))
    _refused("rows must be", q, torch.zeros(5, dtype=BF16))
    _refused("rows must be", q, torch.zeros(1, 2, 3, 4, dtype=BF16))
    _refused("rows must be", q, torch.zeros(3, 0, dtype=BF16))
    _refused("rows must be", q, torch.empty(1, (1 << 17) + 1, dtype=BF16))
    _refused("contiguous last", q, torch.zeros(5, 3, dtype=BF16).t())
    _refused("Inference only", q, torch.zeros(3, 5, dtype=BF16, requires_grad=True))
    with torch.no_grad():
        _refused(ON_DEVICE, q, torch.zeros(3, 5, dtype=BF16, requires_grad=True))
    _refused("nonempty", f.quantize_weight, torch.zeros(3, 2, 5, dtype=BF16))
    _refused("nonempty", f.quantize_weight, torch.zeros(0, 5, dtype=BF16))


def test_adaln_refusals():
    def call(match, **over):
        a = dict(x=torch.zeros(2, 3, 64, dtype=BF16), shift=torch.zeros(2, 64, dtype=BF16),
                 scale=torch.zeros(2, 64, dtype=BF16))
        _refused(match, f.adaln_quantize, **{**a, **over})

    x, v = torch.zeros(2, 3, 64, dtype=BF16), torch.zeros(2, 64, dtype=BF16)
    call(ON_DEVICE)
    call(ON_DEVICE, y=x, gate=v, x_out=x)
    call("x must be", x=torch.zeros(3, 64, dtype=BF16))
    call("bf16 or fp16", x=x.float())
    call("given together", y=x)
    call("given together", gate=v)
    call("only with a residual", x_out=x)
    call("like x", y=x[:, :2], gate=v)
    call("like x", y=x.half(), gate=v)
    call("like x", y=x, gate=v, x_out=x[:1])
    call("shift/scale/gate", shift=v[:1])
    call("shift/scale/gate", scale=v.half())
    call("shift/scale/gate", y=x, gate=torch.zeros(64, 2, dtype=BF16).t())
    call("one batch stride", shift=torch.zeros(2, 128, dtype=BF16)[:, :64])
    call("contiguous last", x=torch.zeros(2, 64, 3, dtype=BF16).transpose(1, 2))
    call("non-overlapping", y=x, gate=v, x_out=torch.zeros(1, 3, 64, dtype=BF16).expand(2, 3, 64))
    call("cannot alias", y=x, gate=v, shift=x.view(6, 64)[:2], scale=x.view(6, 64)[:2], x_out=x)
    call("Inference only", shift=v.clone().requires_grad_())
    # the residual goes over x or y, or apart from both
    h = torch.zeros(2, 8, 64, dtype=BF16)
    call(ON_DEVICE, y=x, gate=v, x=h[:, :3], x_out=h[:, 3:6])
    call(ON_DEVICE, y=h[:, 5:], x=h[:, :3], gate=v, x_out=h[:, 5:])
    call("x itself", y=x, gate=v, x=h[:, :3], x_out=h[:, 2:5])
    call("x itself", y=h[:, 2:5], gate=v, x_out=h[:, :3])
    call("x itself", y=x[:1], gate=v[:1], x=h[:1, :3], x_out=h[:1, 1:4], shift=v[:1], scale=v[:1])
    row = dict(shift=v, scale=v, gate=v)
    t, i = dict(x=h[:, :3], y=x, x_out=h[:, :3], **row), dict(x=h[:, 3:], y=h[:, 3:], x_out=h[:, 3:], **row)
    _refused(ON_DEVICE, f.adaln_quantize_pair, t, i)
    _refused("x itself", f.adaln_quantize_pair, {**t, "x_out": h[:, 3:6]}, i)
    _refused("must lie apart", f.adaln_quantize_pair, {**t, "x": x, "x_out": h[:, :3]}, {**i, "x": x, "y": x, "x_out": h[:, 2:5]})
    a, b = dict(x=x, shift=v, scale=v), dict(x=x[:, :1], shift=v, scale=v)
    _refused(ON_DEVICE, f.adaln_quantize_pair, a, b)
    _refused("one batch", f.adaln_quantize_pair, a, dict(x=x[:1], shift=v[:1], scale=v[:1]))
    _refused("one batch", f.adaln_quantize_pair, a, dict(x=x.half(), shift=v.half(), scale=v.half()))
    _refused("one batch", f.adaln_quantize_pair, a, dict(x=x[..., :32], shift=v[:, :32], scale=v[:, :32]))


def test_linear_refusals():
    x, w, b = _rows(2, 3), _weight(5), torch.zeros(5, dtype=BF16)
    out = torch.zeros(2, 3, 5, dtype=BF16)

    def call(match, x=x, w=w, b=None, **kw):
        _refused(match, f.int8_linear, x, w, b, **kw)

    call(ON_DEVICE)
    call(ON_DEVICE, b=b, out=out, gelu=True)
    call(ON_DEVICE, x=torch.zeros(2, 3, 70, dtype=BF16))
    call("takes 70 features", x=_rows(2, 3, features=71))
    call("as the rows are padded", w=f.Int8Weight(torch.zeros(5, 192, dtype=torch.int8), torch.zeros(5), 70))
    call("contiguous int8", x=x._replace(q=x.q.float()))
    call("contiguous int8", x=x._replace(q=x.q.transpose(0, 1).contiguous().transpose(0, 1)))
    call("contiguous int8", x=x._replace(q=x.q[..., :70].contiguous()))
    call("float32 scale", x=x._replace(scale=x.scale.double()))
    call("float32 scale", x=x._replace(scale=x.scale[:1]))
    call("float32 scale", w=w._replace(scale=torch.zeros(6)))
    call("bf16 or fp16", x=x._replace(dtype=torch.float32))
    call("bias", b=b[:4])
    call("bias", b=b.half())
    call("bias", b=torch.zeros(10, dtype=BF16)[::2])
    call("rows' dtype", out=out.half())
    call("leading dimensions", out=out[:, :2])
    call("as the rows are padded", out=torch.zeros(2, 3, 6, dtype=BF16))
    call("contiguous last", out=torch.zeros(2, 5, 3, dtype=BF16).transpose(1, 2))
    call("non-overlapping", out=torch.zeros(2, 1, 5, dtype=BF16).expand(2, 3, 5))
    call("non-overlapping", out=torch.zeros(100, dtype=BF16).as_strided((2, 3, 5), (5, 5, 1)))
    shared = torch.zeros(64, dtype=BF16)
    call("cannot alias", b=shared[3:8], out=shared[:30].view(2, 3, 5))
    call("Inference only", b=b.clone().requires_grad_())
    call("Inference only", x=torch.zeros(2, 3, 70, dtype=BF16, requires_grad=True))
    buf = torch.zeros(2, 9, 12, dtype=BF16)
    for first, second in ((buf[:, :3, :5], buf[:, 3:6, :5]), (buf[:, :3, :5], buf[:, :3, 5:10]), (buf[:, 3:6, 7:], buf[:, :3, 7:])):
        _refused(ON_DEVICE, f.int8_linear_pair, dict(x=x, weight=w, out=first), dict(x=x, weight=w, out=second))
    for first, second in ((buf[:, :3, :5], buf[:, 2:5, :5]), (buf[:, :3, :5], buf[:, :3, 4:9]), (out, out)):
        _refused("lie apart", f.int8_linear_pair, dict(x=x, weight=w, out=first), dict(x=x, weight=w, out=second))
    _refused("cannot alias", f.int8_linear_pair, dict(x=x, weight=w, out=shared[:30].view(2, 3, 5)),
             dict(x=x, weight=w, bias=shared[10:15]))
    a = dict(x=x, weight=w, bias=b)
    _refused(ON_DEVICE, f.int8_linear_pair, a, dict(x=_rows(2, 9), weight=w))
    _refused("must share", f.int8_linear_pair, a, dict(x=_rows(1, 9), weight=w))
    _refused("must share", f.int8_linear_pair, a, dict(x=_rows(2, 9), weight=_weight(6)))
    _refused("must share", f.int8_linear_pair, a, dict(x=_rows(2, 9, features=200), weight=_weight(5, 200)))
    _refused("must share", f.int8_linear_pair, a, dict(x=_rows(2, 9, dtype=FP16), weight=w))


def test_qkv_refusals():
    H, T, n = 2, 4, 6
    text, image, w, norm = _rows(3, T), _rows(3, n), _weight(3 * H * 128), torch.zeros(128, dtype=BF16)
    table = torch.zeros(T + n, 128)

    def call(match, text=text, image=image, **over):
        _refused(match, f.int8_qkv, text, image, **{**dict(heads=H, weights=(w, w)), **over})

    call(ON_DEVICE)
    call(ON_DEVICE, norms=((norm, None), (None, norm)), cos=table, sin=table, biases=(None, torch.zeros(768, dtype=BF16)))
    call(ON_DEVICE, text=None, weights=(None, w))
    call("share features", text=_rows(3, T, features=80))
    call("share features", text=_rows(3, T, dtype=FP16))
    call("rows' features", weights=(w, _weight(768, 71)))
    call("rows' features", weights=(_weight(768, 71), w))
    call("nonempty", image=_rows(3, 0))
    call("nonempty", image=_rows(n), text=None)
    call("one batch", text=_rows(2, T))
    call("as the rows are padded", heads=3)
    call("norm weights", norms=((norm[:64], norm), (norm, norm)))
    call("norm weights", norms=((norm, norm), (norm, norm.float())))
    call("bias", biases=(torch.zeros(767, dtype=BF16), None))
    call("given together", cos=table)
    call("cos/sin", cos=table[1:], sin=table[1:])
    call("cos/sin", cos=table.half(), sin=table.half())
    call("rows' dtype", out=torch.zeros(3, 3, T + n, H, 128, dtype=FP16))
    call(r"\[3, B, N, heads, 128\]", out=torch.zeros(2, 3, T + n, H, 128, dtype=BF16))
    call("text rows and then", out=torch.zeros(3, 3, T + n + 1, H, 128, dtype=BF16))
    call("contiguous heads", out=torch.zeros(3, 3, T + n, H, 256, dtype=BF16)[..., :128])
    call("non-overlapping", out=torch.zeros(1, 3, T + n, H, 128, dtype=BF16).expand(3, -1, -1, -1, -1))
    call("Inference only", norms=((norm, norm.clone().requires_grad_()), (norm, norm)))


def test_missing_gradients_are_refused_by_transforms():
    x, w = _rows(2, 3), _weight(5)
    with pytest.raises(Exception):
        torch.func.grad(lambda b: f.int8_linear(x, w, b).float().sum())(torch.zeros(5, dtype=BF16))


# ------------------------------------------------------------------ C entry points
def _einval(match, name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1 and match in _lib.last_error(), _lib.last_error()


def test_entry_points_reject_before_any_launch():
    P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32

    def rows(x=16, bs=0, rs=64, batch=1, rows=4, features=60, padded=64, dtype=0, q=256, scale=512):
        return (x, bs, rs, batch, rows, features, padded, dtype, q, scale, None)

    for match, over in (("null", dict(x=None)), ("null", dict(scale=None)), ("positive", dict(rows=0)),
                        ("2^31", dict(batch=1 << 16, rows=1 << 16)), ("too many", dict(batch=2, rows=1 << 25)),
                        ("too many", dict(rows=1 << 24, features=3073, padded=3136)), ("features", dict(features=0)),
                        ("features", dict(features=(1 << 17) + 1)), ("padded", dict(padded=63)), ("padded", dict(features=65)),
                        ("dtype", dict(dtype=2)), ("aligned", dict(x=17)), ("aligned", dict(q=264)), ("strides", dict(rs=-1))):
        _einval(match, "hb_int8_rows", *rows(**over))

    def adaln(count=1, batch=1, rows=(4,), hidden=64, padded=64, dtype=0, eps=1e-6, pointers=(16, None, None, None, 16, 16, 16, 16),
              strides=(64,) * 8):
        return (count, batch, (I32 * 2)(*rows), hidden, padded, dtype, eps, (P * 16)(*pointers), (I64 * 16)(*strides), None)

    p = (16, None, None, None, 16, 16, 16, 16)
    for match, over in (("count", dict(count=3)), ("hidden", dict(hidden=60)), ("hidden", dict(hidden=8200, padded=8256)),
                        ("padded", dict(padded=72)), ("dtype", dict(dtype=9)), ("eps", dict(eps=0.0)), ("positive", dict(batch=0)),
                        ("too many", dict(batch=4, rows=(1 << 24,))),
                        ("null", dict(pointers=(None,) + p[1:])), ("given together", dict(pointers=(16, 16) + p[2:])),
                        ("residual", dict(pointers=(16, None, None, 16) + p[4:])), ("16-byte", dict(pointers=(24,) + p[1:])),
                        ("4-byte", dict(pointers=p[:7] + (18,))), ("multiples of 8", dict(strides=(4,) + (64,) * 7))):
        _einval(match, "hb_int8_adaln", *adaln(**over))

    def linear(count=1, batch=1, rows=(4, 4), columns=40, padded=64, dtype=0, gelu=0, pointers=(256, 256, 256, 256, None, 256),
               strides=(0, 40, 0, 40)):
        return (count, batch, (I32 * 2)(*rows), columns, padded, dtype, gelu, (P * 12)(*pointers), (I64 * 4)(*strides), None)

    def few(x=16, bs=0, rs=64, batch=1, rows=4, features=60, columns=40, padded=64, dtype=0, gelu=0, w=256, ws=256, bias=None,
            out=256, ob=0, on=40):
        return (x, bs, rs, batch, rows, features, columns, padded, dtype, gelu, w, ws, bias, out, ob, on, None)

    for match, over in (("null", dict(x=None)), ("null", dict(w=None)), ("null", dict(out=None)), ("positive", dict(rows=0)),
                        ("32 rows", dict(rows=33)), ("32 rows", dict(batch=8, rows=5)), ("8 features", dict(features=7)),
                        ("padded", dict(padded=72)), ("padded", dict(features=65)), ("padded", dict(padded=16448)),
                        ("16384 values", dict(rows=3, features=8000, padded=8000)), ("columns", dict(columns=0)),
                        ("dtype", dict(dtype=2)), ("gelu", dict(gelu=2)), ("aligned", dict(w=264)), ("aligned", dict(x=17)),
                        ("aligned", dict(ws=258)), ("strides", dict(on=-1))):
        _einval(match, "hb_int8_linear_rows", *few(**over))

    p = (256, 256, 256, 256, None, 256)
    for match, over in (("count", dict(count=0)), ("columns", dict(columns=0)), ("padded", dict(padded=72)),
                        ("padded", dict(padded=1 << 18)), ("dtype", dict(dtype=2)), ("gelu", dict(gelu=2)),
                        ("positive", dict(rows=(0, 4))), ("null", dict(pointers=p[:3] + (None,) + p[4:])),
                        ("16-byte", dict(pointers=(264,) + p[1:])), ("4-byte", dict(pointers=(256, 258) + p[2:])),
                        ("2-byte", dict(pointers=p[:5] + (257,))), ("non-negative", dict(strides=(0, -40, 0, 0))),
                        ("null", dict(count=2, pointers=p))):
        _einval(match, "hb_int8_linear", *linear(**over))

    def qkv(batch=1, text=0, tokens=4, heads=2, padded=64, dtype=0, eps=1e-6, pointers=(None,) * 7 + (256,) * 4 + (None,) * 3,
            cos=None, sin=None, out=256, strides=(4 * 256, 4 * 256, 256)):
        return (batch, text, tokens, heads, padded, dtype, eps, (P * 14)(*pointers), cos, sin, out, *strides, None)

    for match, over in (("tokens", dict(tokens=0)), ("tokens", dict(text=4)), ("heads", dict(heads=0)), ("eps", dict(eps=0.0)),
                        ("given together", dict(cos=256)), ("16-byte", dict(out=264)), ("multiples of 8", dict(strides=(4, 8, 8))),
                        ("null", dict(text=1)), ("null", dict(out=None)), ("padded", dict(padded=65))):
        _einval(match, "hb_int8_qkv", *qkv(**over))


# ------------------------------------------------------------------ the oracle
def test_oracle_quantize():
    x = torch.tensor([[1.0, -0.5, 0.25, 0.0], [0.0, 0.0, 0.0, 0.0]], dtype=BF16)
    q, s, _ = O.quantize(x)
    assert q.tolist() == [[127, -64, 32, 0], [0, 0, 0, 0]]  # 63.5 to even, 31.75
    assert s.tolist() == [1 / 127, 0.0]


def test_oracle_linear_and_gelu():
    q = torch.tensor([[1, 2], [-3, 4]], dtype=torch.int8)
    w = torch.tensor([[5, -6]], dtype=torch.int8)
    p, d = O.linear(q, torch.tensor([0.5, 2.0]), w, torch.tensor([0.25]), torch.tensor([1.0], dtype=BF16))
    assert p.flatten().tolist() == [-7 * 0.125 + 1, -39 * 0.5 + 1]
    v = torch.linspace(-6, 6, 101, dtype=torch.float64)
    g, _ = O.gelu(v, torch.zeros_like(v))
    assert torch.allclose(g, torch.nn.functional.gelu(v, approximate="tanh"), rtol=1e-12, atol=1e-15)


def test_oracle_adaln_and_qkv():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 16, generator=gen, dtype=torch.float64)
    sh, sc, g = (torch.randn(2, 16, generator=gen, dtype=torch.float64) for _ in range(3))
    y = torch.randn(2, 3, 16, generator=gen, dtype=torch.float64)
    m, dm, r, _ = O.adaln(x, sh, sc, y, g)
    ref = torch.nn.functional.layer_norm(x + g[:, None] * y, (16,), eps=1e-6) * (1 + sc[:, None]) + sh[:, None]
    assert torch.allclose(m, ref, rtol=1e-12) and (dm >= 0).all()
    p = torch.randn(1, 3, 3 * 2 * 128, generator=gen, dtype=torch.float64)
    angle = torch.rand(3, 64, generator=gen, dtype=torch.float64) * 2 * math.pi
    w = torch.randn(128, generator=gen, dtype=torch.float64)
    c, s = (t.repeat_interleave(2, 1) for t in (angle.cos(), angle.sin()))
    (q, _), _, (v, _) = O.qkv(p, torch.zeros_like(p), 2, w.expand(3, -1), None, c, s)
    a = p.view(1, 3, 3, 2, 128)
    n = a[:, :, 0] / (a[:, :, 0].square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    z = torch.view_as_complex(n.unflatten(-1, (64, 2)).contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    assert torch.allclose(q, torch.view_as_real(z).flatten(-2), rtol=1e-10, atol=1e-12)
    assert torch.equal(v, a[:, :, 2])
