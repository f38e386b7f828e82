"""The 8-bit linear layers on the GPU against their definition in 64 bits (oracle/int8_ops.py).

8-bit rows are exact, so they are compared for equality (quantize_rows), or held to half a step plus the
fp32 error of the value (adaln_quantize).  Products are held to their fp32 error, derived in the oracle,
and one rounding to the output's type.
"""

import pytest
import torch

from hilberta_amd.flux_int8 import (
    Int8Rows,
    Int8Weight,
    adaln_quantize,
    adaln_quantize_pair,
    int8_linear,
    int8_linear_pair,
    int8_qkv,
    padded_features,
    quantize_rows,
    quantize_weight,
)
from hilberta_amd.flux_inputs import rotary_tables
from oracle import int8_ops as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=BF16, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def _int8(gen, rows, features, scale=0.01):
    """8-bit rows over the whole range, zeros in the padding, and scales around ``scale``."""
    lead = (rows,) if isinstance(rows, int) else tuple(rows)
    q = torch.zeros(*lead, padded_features(features), dtype=torch.int8, device="cuda")
    q[..., :features] = torch.randint(-127, 128, (*lead, features), generator=gen, device="cuda").to(torch.int8)
    s = (torch.rand(*lead, generator=gen, device="cuda") + 0.5) * scale
    return q, s


def _rows(gen, lead, features, dtype=BF16):
    return Int8Rows(*_int8(gen, lead, features), features, dtype)


def _weight(gen, columns, features):
    return Int8Weight(*_int8(gen, columns, features, 0.01 * features**-0.5), features)


def _check_linear(got, x, w, bias, gelu=False, what=""):
    p, d = O.linear(x.q, x.scale, w.q, w.scale, bias)
    if gelu:
        p, d = O.gelu(p, d)
    O.held(got, p, d, what)


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,features", [(1, 1), (3, 7), (5, 63), (2, 64), (4, 65), (7, 511), (9, 648), (3, 1000),
                                           (300, 777), (6, 3072), (5, 4097), (3, 12288), (2, 15360), (2, 20001)])
def test_rows_are_exact(rows, features, dtype):
    gen = _gen(rows * features)
    x = _randn(gen, rows, features, dtype=dtype)
    x[0, features // 2] = 4.0 * x[0].abs().max()  # quarters and halves of it are ties
    x[0, :features // 2] = (x[0, :features // 2] * 0 + x[0, features // 2] / 2)
    r = quantize_rows(x)
    q, scale, _ = O.quantize(x)
    assert r.q.shape == (rows, padded_features(features)) and r.features == features and r.dtype == dtype
    assert torch.equal(r.q[:, :features].long(), q)
    assert not r.q[:, features:].any()
    assert ((r.scale.double() - scale).abs() <= O.U * scale).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_value_rounds_exactly(dtype):
    """Every 16-bit value up to a row's top, for several tops."""
    bits = torch.arange(0x8000, dtype=torch.int32).to(torch.int16).view(dtype)
    bits = bits[torch.isfinite(bits)].cuda()
    for top in (1.0, 1.9921875, 0.3359375, 447.0, 2.0**-13):
        top = torch.tensor(top).to(dtype).item()
        x = bits[bits <= top]
        x = torch.cat([x, -x, x.new_full((1,), top)])[None]
        r = quantize_rows(x)
        q, _, _ = O.quantize(x)
        assert torch.equal(r.q[:, :x.shape[1]].long(), q), top


def test_rows_of_little_nothing_and_not_numbers():
    tiny = torch.full((1, 70), 2.0**-133, dtype=BF16, device="cuda")  # the smallest of the type
    tiny[0, 3] = -tiny[0, 3] * 2
    r = quantize_rows(tiny)
    assert r.q[0, 3] == -127 and (r.q[0, :3] == 64).all()  # 63.5, a tie, to even
    small = torch.full((1, 70), 2.0**-70, dtype=BF16, device="cuda")
    assert (quantize_rows(small).q[0, :70] == 127).all()
    huge = torch.full((1, 70), 3e38, dtype=BF16, device="cuda")
    assert (quantize_rows(huge).q[0, :70] == 127).all()
    zero = quantize_rows(torch.zeros(2, 70, dtype=FP16, device="cuda"))
    assert not zero.q.any() and not zero.scale.any()
    for bad in (float("inf"), float("-inf"), float("nan")):
        for dtype in (BF16, FP16):
            x = torch.ones(3, 70, dtype=dtype, device="cuda")
            x[1, 69] = bad
            r = quantize_rows(x)
            assert torch.isnan(r.scale[1]) and torch.isfinite(r.scale[[0, 2]]).all()
            assert (r.q[[0, 2], :70] == 127).all()
            w = _weight(_gen(1), 40, 70)
            out = int8_linear(r, w)
            assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()


def test_rows_larger_than_the_caches():
    """What is read past the caches is the same."""
    gen = _gen(5)
    for features in (1000, 9000):
        x = _randn(gen, (1 << 27) // features, features, dtype=FP16)
        r = quantize_rows(x)
        assert all(torch.equal(r.q[at:at + 1000, :features].long(), O.quantize(x[at:at + 1000])[0])
                   for at in range(0, len(x), 1000))
        assert not r.q[:, features:].any()


def test_adaln_larger_than_the_caches():
    gen = _gen(6)
    for C in (640, 3072):
        M = (1 << 26) // C
        x, y, mod = _randn(gen, 1, M, C), _randn(gen, 1, M, C), _randn(gen, 1, 3 * C, std=0.3)
        shift, scale, gate = mod.chunk(3, 1)
        out = torch.empty_like(x)
        r = adaln_quantize(x, shift, scale, y=y, gate=gate, x_out=out)
        for at in range(0, M, 5000):
            part, one = slice(at, at + 5000), torch.empty_like(x[:, at:at + 5000])
            few = adaln_quantize(x[:, part], shift, scale, y=y[:, part], gate=gate, x_out=one)
            assert torch.equal(few.q, r.q[:, part]) and torch.equal(few.scale, r.scale[:, part]) and torch.equal(one, out[:, part])


def test_rows_by_strides():
    gen = _gen(5)
    big = _randn(gen, 3, 50, 400)
    for x in (big[:, 7:30, 1:334], big[1:, ::2, :64], big[:, :, 8:9], big[0, 3:4].expand(6, 400),
              big[:1].expand(4, 50, 400), big.transpose(0, 1)[:, :, :128]):
        r = quantize_rows(x)
        assert torch.equal(r.q[..., :x.shape[-1]].long(), O.quantize(x)[0])
    with pytest.raises(ValueError, match="contiguous last"):
        quantize_rows(big.transpose(1, 2))
    empty = quantize_rows(big[:, :0])
    assert empty.q.shape == (3, 0, 448) and empty.scale.shape == (3, 0)


# ------------------------------------------------------------------ AdaLN
def _check_adaln(rows, x, shift, scale, y=None, gate=None, x_out=None):
    hidden = x.shape[-1]
    m, dm, r, dr = O.adaln(x, shift, scale, y, gate)
    _, _, quotient = O.quantize(m)
    top = m.abs().amax(-1, keepdim=True)
    dtop = dm.amax(-1, keepdim=True)
    slack = 127 * (dm / top + m.abs() * dtop / top**2) * 1.01 + 127 * 4 * O.U
    assert ((rows.q[..., :hidden].double() - quotient).abs() <= 0.5 + slack).all()
    assert slack.max() < 0.1  # (the comparison says something)
    assert not rows.q[..., hidden:].any()
    assert ((rows.scale.double() - top[..., 0] / 127).abs() <= (dtop[..., 0] + 2 * O.U * top[..., 0]) / 127).all()
    if x_out is not None:
        O.held(x_out, r, dr, "residual")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("batch,rows,hidden", [(1, 1, 8), (2, 3, 72), (1, 64, 512), (3, 5, 520), (2, 33, 1024),
                                               (1, 7, 1544), (2, 130, 3072), (1, 9, 4096), (1, 5, 5120), (1, 3, 8192)])
def test_adaln(batch, rows, hidden, dtype):
    gen = _gen(hidden + rows)
    x, y = _randn(gen, batch, rows, hidden, dtype=dtype), _randn(gen, batch, rows, hidden, dtype=dtype)
    mod = _randn(gen, batch, 3 * hidden, dtype=dtype, std=0.3)
    shift, scale, gate = mod.chunk(3, 1)
    _check_adaln(adaln_quantize(x, shift, scale), x, shift, scale)
    _check_adaln(adaln_quantize(x, shift, scale, y=y, gate=gate), x, shift, scale, y, gate)
    before, x_out = x.clone(), x  # in place
    got = adaln_quantize(x, shift, scale, y=y, gate=gate, x_out=x_out)
    _check_adaln(got, before, shift, scale, y, gate, x_out)


def test_adaln_of_row_ranges_in_one_launch():
    gen = _gen(11)
    B, T, n, C = 2, 5, 70, 512
    h = _randn(gen, B, T + n, C)
    y = _randn(gen, B, T + n, C)
    mod = _randn(gen, B, 6 * C, std=0.3)
    sh, sc, g, sh2, sc2, g2 = mod.chunk(6, 1)
    out = torch.full((B, T + n + 2, C), 7.0, dtype=BF16, device="cuda")
    image, text = adaln_quantize_pair(
        dict(x=h[:, T:], shift=sh, scale=sc, y=y[:, T:], gate=g, x_out=out[:, T:T + n]),
        dict(x=h[:, :T], shift=sh2, scale=sc2, y=y[:, :T], gate=g2, x_out=out[:, :T]))
    _check_adaln(image, h[:, T:], sh, sc, y[:, T:], g, out[:, T:T + n])
    _check_adaln(text, h[:, :T], sh2, sc2, y[:, :T], g2, out[:, :T])
    assert (out[:, T + n:] == 7).all()
    plain = adaln_quantize_pair(dict(x=h[:, T:], shift=sh, scale=sc), dict(x=h[:, :T], shift=sh2, scale=sc2))
    for got, one in zip(plain, (adaln_quantize(h[:, T:], sh, sc), adaln_quantize(h[:, :T], sh2, sc2))):
        assert torch.equal(got.q, one.q) and torch.equal(got.scale, one.scale)


def test_adaln_of_one_image_for_a_batch_and_bad_rows():
    gen = _gen(12)
    x = _randn(gen, 1, 9, 512).expand(3, 9, 512)
    mod = _randn(gen, 1, 1024, std=0.3).expand(3, 1024)
    shift, scale = mod.chunk(2, 1)
    _check_adaln(adaln_quantize(x, shift, scale), x, shift, scale)
    x = _randn(gen, 1, 3, 512)
    x[0, 1, 500] = float("inf")
    r = adaln_quantize(x, shift[:1], scale[:1])
    assert torch.isnan(r.scale[0, 1]) and torch.isfinite(r.scale[0, ::2]).all()
    flat = torch.full((1, 2, 512), 3.0, dtype=BF16, device="cuda")  # no variance: the shift alone
    got = adaln_quantize(flat, shift[:1], scale[:1])  # (sums of threes are exact, and so are the differences)
    assert torch.equal(got.q.long(), O.quantize(shift[:1, None].expand(1, 2, 512))[0])


# ------------------------------------------------------------------ products
ROWS = [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 513, 700]


@pytest.mark.parametrize("rows", ROWS)
def test_linear_over_rows(rows):
    gen = _gen(rows)
    for features, columns, dtype, bias, gelu in ((192, 128, BF16, True, False), (1000, 777, FP16, True, True),
                                                 (64, 33, BF16, False, False), (2112, 264, FP16, False, False)):
        x, w = _rows(gen, rows, features, dtype), _weight(gen, columns, features)
        b = _randn(gen, columns, dtype=dtype) if bias else None
        _check_linear(int8_linear(x, w, b, gelu=gelu), x, w, b, gelu, f"{rows} x {features} x {columns}")


@pytest.mark.parametrize("columns", [1, 7, 8, 16, 31, 32, 64, 100, 128, 129, 136, 255, 256, 257, 300, 520, 1030])
@pytest.mark.parametrize("rows", [1, 20, 77, 384, 520])
def test_linear_over_columns(rows, columns):
    gen = _gen(columns)
    x, w = _rows(gen, rows, 320), _weight(gen, columns, 320)
    b = _randn(gen, columns)
    _check_linear(int8_linear(x, w, b), x, w, b, False, f"{columns} columns")


@pytest.mark.parametrize("features", [1, 16, 63, 64, 65, 128, 192, 200, 256, 320, 448, 512, 1024, 3072, 4100, 12288])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_over_features(rows, features):
    gen = _gen(features)
    x, w = _rows(gen, rows, features), _weight(gen, 272, features)
    _check_linear(int8_linear(x, w), x, w, None, False, f"{features} features")


@pytest.mark.parametrize("rows,features,columns", [(1, 3072, 18432), (13, 3072, 9216), (77, 4096, 3072),
                                                   (512, 12288, 3072), (1000, 3072, 3072), (4096, 3072, 3072),
                                                   (2500, 1024, 9000)])
def test_linear_of_real_sizes(rows, features, columns):
    gen = _gen(rows)
    x, w = _rows(gen, rows, features), _weight(gen, columns, features)
    b = _randn(gen, columns)
    _check_linear(int8_linear(x, w, b, gelu=True), x, w, b, True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,features,columns", [(1, 1122, 53), (2739, 1141, 135), (135, 1110, 3307), (335, 1106, 2721),
                                                   (2703, 1091, 485), (833, 1098, 3489), (14, 1122, 256), (700, 1200, 3010)])
def test_linear_over_tiles(rows, features, columns, dtype):
    """Each shape of tile, its ring of stages walked past its end, ragged on every side."""
    gen = _gen(rows)
    x, w = _rows(gen, rows, features, dtype), _weight(gen, columns, features)
    b = _randn(gen, columns, dtype=dtype)
    for gelu in (False, True):
        _check_linear(int8_linear(x, w, b, gelu=gelu), x, w, b, gelu)


@pytest.mark.parametrize("features", [1400, 15360])
def test_last_rows_apart(features):
    """Tiles that fill whole rounds of the CUs, and the rows after them: 66 x 12 of 256 x 256."""
    gen = _gen(features)
    M, N = 16896 - 77, 12 * 256 - 8
    x, w = _rows(gen, (3, M // 3), features), _weight(gen, N, features)
    out, again = (int8_linear(x, w) for _ in range(2))
    assert torch.equal(out, again)
    flat = Int8Rows(x.q.flatten(0, 1), x.scale.flatten(), features, BF16)
    for at in (slice(0, 40), slice(16300, 16420), slice(M // 3 * 3 - 40, M)):
        part = Int8Rows(flat.q[at], flat.scale[at], features, BF16)
        _check_linear(out.flatten(0, 1)[at], part, w, None)
    assert torch.equal(out.flatten(0, 1)[16000:], int8_linear(flat._replace(q=flat.q[16000:], scale=flat.scale[16000:]), w))


def test_last_rows_of_the_second_set_apart():
    gen = _gen(17)
    K, N = 1400, 3064
    sets = [dict(x=_rows(gen, (2, rows), K), weight=_weight(gen, N, K), bias=_randn(gen, N)) for rows in (256, 8192 - 77)]
    for out, s in zip(int8_linear_pair(*sets), sets):
        assert torch.equal(out, torch.cat([int8_linear(s["x"]._replace(q=s["x"].q[b:b + 1], scale=s["x"].scale[b:b + 1]),
                                                       s["weight"], s["bias"]) for b in range(2)]))
        for at in (slice(0, 30), slice(-30, None)):
            x = Int8Rows(s["x"].q[1, at], s["x"].scale[1, at], K, BF16)
            _check_linear(out[1, at], x, s["weight"], s["bias"])


@pytest.mark.parametrize("offset", range(8))
def test_linear_into_rows_that_start_anywhere(offset):
    """Output rows at every alignment of whole elements, odd strides among them; what is around them stays."""
    gen = _gen(offset)
    for M, K, N in ((50, 192, 100), (130, 192, 264), (40, 64, 7)):
        x, w = _rows(gen, M, K), _weight(gen, N, K)
        want = int8_linear(x, w)
        for pad in (8, 9, 10):
            buf = torch.full((M, N + pad + offset), 5.0, dtype=BF16, device="cuda")
            int8_linear(x, w, out=buf[:, offset:offset + N])
            assert torch.equal(buf[:, offset:offset + N], want)
            assert (buf[:, :offset] == 5).all() and (buf[:, offset + N:] == 5).all()


def test_linear_takes_16_bit_rows():
    gen = _gen(3)
    x, weight, b = _randn(gen, 2, 50, 333, dtype=FP16), _randn(gen, 90, 333, dtype=FP16, std=0.05), _randn(gen, 90, dtype=FP16)
    w = quantize_weight(weight)
    assert torch.equal(w.q[:, :333].long(), O.quantize(weight)[0])
    rows = quantize_rows(x)
    out = int8_linear(x, w, b)
    assert out.shape == (2, 50, 90) and out.dtype == FP16
    assert torch.equal(out, int8_linear(rows, w, b))
    _check_linear(out, rows, w, b)
    # near the 16-bit layer: each of the two roundings to 8 bits is off by half a step of the row's top / 127
    ref = torch.nn.functional.linear(x.double(), weight.double(), b.double())
    top = lambda t: t.double().abs().amax(-1)  # noqa: E731
    step = (x.double().abs().sum(-1)[..., None] * top(weight) / 254 + weight.double().abs().sum(-1) * top(x)[..., None] / 254
            + 333 * top(x)[..., None] * top(weight) / 254**2)
    O.held(out, ref, step * 1.01)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lead,features,columns", [((1,), 8, 1), ((1,), 3072, 18432), ((1,), 16384, 100), ((2,), 8192, 33),
                                                   ((2,), 8129, 65), ((32,), 512, 300), ((31,), 500, 129), ((3, 2), 777, 64),
                                                   ((1, 5), 2049, 4100), ((4, 8), 9, 40), ((2, 1), 64, 12290),
                                                   ((7,), 2111, 13000), ((1,), 65, 31), ((33,), 100, 50), ((2,), 8193, 40)])
def test_linear_of_a_few_16_bit_rows(lead, features, columns, dtype):
    """One launch gives what two do, to the bit: up to 32 rows and 16384 values, and past that."""
    gen = _gen(features)
    big = _randn(gen, *lead, features + 11, dtype=dtype)
    b = _randn(gen, columns, dtype=dtype)
    w = _weight(gen, columns, features)
    for x in (big[..., :features].contiguous(), big[..., 3:features + 3]):
        rows = quantize_rows(x)
        for gelu, bias in ((False, None), (True, b)):
            got = int8_linear(x, w, bias, gelu=gelu)
            assert got.shape == (*lead, columns) and torch.equal(got, int8_linear(rows, w, bias, gelu=gelu))
    _check_linear(got, rows, w, b, True)


def test_a_few_bad_rows():
    gen = _gen(4)
    x = _randn(gen, 5, 300)
    x[1] = 0
    x[2, 7], x[3, 299], x[4, 0] = float("inf"), float("nan"), 3e38
    w, b = _weight(gen, 70, 300), _randn(gen, 70)
    got = int8_linear(x, w, b)
    assert torch.equal(got[:2], int8_linear(quantize_rows(x[:2]), w, b)) and torch.equal(got[1], b)
    assert torch.isnan(got[2:4]).all() and torch.equal(got[4], int8_linear(quantize_rows(x), w, b)[4])
    empty = int8_linear(x[:0], w, b)
    assert empty.shape == (0, 70)


def test_largest_sums():
    """Every product 127 * 127 over 2^17 features: the sum fits 32 bits."""
    K = 1 << 17
    x = Int8Rows(torch.full((2, K), 127, dtype=torch.int8, device="cuda"), torch.full((2,), 1e-5, device="cuda"), K, BF16)
    w = Int8Weight(torch.full((3, K), -128, dtype=torch.int8, device="cuda"), torch.full((3,), 1e-5, device="cuda"), K)
    _check_linear(int8_linear(x, w), x, w, None)


@pytest.mark.parametrize("rows", [3, 40, 150, 600])
def test_linear_into_views(rows):
    """Row ranges and column blocks of a larger buffer, at addresses of every alignment; the rest stays."""
    gen = _gen(rows)
    x, w = _rows(gen, (2, rows), 192), _weight(gen, 136, 192)
    want = int8_linear(x, w)
    _check_linear(want, x, w, None)
    for lead, first, width in ((5, 0, 136), (0, 8, 160), (3, 1, 139), (2, 24, 168), (1, 3, 256)):
        buf = torch.full((2, rows + lead + 1, width), 5.0, dtype=BF16, device="cuda")
        view = buf[:, lead:lead + rows, first:first + 136]
        assert int8_linear(x, w, out=view) is view
        assert torch.equal(view, want)
        view.fill_(5.0)
        assert (buf == 5).all()
    flat = int8_linear(Int8Rows(x.q[1], x.scale[1], 192, BF16), w)
    assert torch.equal(flat, want[1])


@pytest.mark.parametrize("sizes", [(5, 40), (64, 300), (512, 77), (1, 1), (130, 1000)])
def test_linear_pair(sizes):
    gen = _gen(sizes[0])
    B, K, N = 2, 448, 264
    sets = [dict(x=_rows(gen, (B, n), K), weight=_weight(gen, N, K), bias=_randn(gen, N)) for n in sizes]
    joint = torch.full((B, sum(sizes), N), 5.0, dtype=BF16, device="cuda")
    sets[0]["out"], sets[1]["out"] = joint[:, :sizes[0]], joint[:, sizes[0]:]
    for got, s in zip(int8_linear_pair(*sets, gelu=True), sets):
        _check_linear(got, s["x"], s["weight"], s["bias"], True)
        assert got is s["out"]


def test_linear_of_no_rows():
    w = _weight(_gen(1), 40, 64)
    assert int8_linear(torch.empty(0, 64, dtype=BF16, device="cuda"), w).shape == (0, 40)
    assert int8_linear(torch.empty(2, 0, 64, dtype=BF16, device="cuda"), w).shape == (2, 0, 40)


# ------------------------------------------------------------------ Q/K/V
def _qkv_set(gen, B, rows, K, heads, dtype, bias=True, norms=True):
    N = 3 * heads * 128
    return dict(x=_rows(gen, (B, rows), K, dtype), w=_weight(gen, N, K), b=_randn(gen, N, dtype=dtype) if bias else None,
                q=_randn(gen, 128, dtype=dtype) if norms else None, k=_randn(gen, 128, dtype=dtype) if norms else None)


def _check_qkv(out, sets, heads, cos, sin):
    p = [O.linear(s["x"].q, s["x"].scale, s["w"].q, s["w"].scale, s["b"]) for s in sets]
    p, d = torch.cat([a for a, _ in p], 1), torch.cat([a for _, a in p], 1)
    norms = [None if sets[-1][n] is None else torch.cat([s[n].expand(s["x"].q.shape[1], -1) for s in sets]) for n in "qk"]
    for plane, (value, bound) in enumerate(O.qkv(p, d, heads, *norms, cos, sin)):
        O.held(out[plane], value, bound, "QKV"[plane])


def _tables(T, n):
    at = torch.arange(n, device="cuda")
    ids = torch.zeros(T + n, 3, device="cuda")
    ids[T:, 1], ids[T:, 2] = at // 7, at % 7
    return rotary_tables(ids)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,n,heads,K", [(1, 0, 1, 1, 64), (1, 0, 1, 24, 3072), (2, 1, 1, 3, 128), (1, 5, 30, 2, 200),
                                           (3, 77, 51, 5, 648), (1, 130, 260, 4, 512), (2, 0, 129, 3, 320),
                                           (1, 33, 600, 2, 1024), (1, 512, 1024, 24, 3072), (1, 4, 13, 1, 1126),
                                           (1, 163, 97, 9, 1110), (2, 3, 193, 11, 1167), (1, 145, 1170, 12, 1102)])
def test_qkv(B, T, n, heads, K, dtype):
    gen = _gen(n + heads)
    sets = ([_qkv_set(gen, B, T, K, heads, dtype)] if T else []) + [_qkv_set(gen, B, n, K, heads, dtype)]
    cos, sin = _tables(T, n)
    t, i = (sets[0] if T else None), sets[-1]
    out = int8_qkv(t and t["x"], i["x"], heads=heads, weights=(t and t["w"], i["w"]), biases=(t and t["b"], i["b"]),
                   norms=((t and t["q"], i["q"]), (t and t["k"], i["k"])), cos=cos, sin=sin)
    assert out.shape == (3, B, T + n, heads, 128) and out.dtype == dtype and out.is_contiguous()
    _check_qkv(out, sets, heads, cos, sin)


@pytest.mark.parametrize("B,T,n", [(1, 0, 14587), (1, 500, 14060), (2, 250, 7030)])
def test_qkv_last_rows_apart(B, T, n):
    gen = _gen(n)
    heads, K = 24, 1400
    sets = ([_qkv_set(gen, B, T, K, heads, BF16)] if T else []) + [_qkv_set(gen, B, n, K, heads, BF16)]
    cos, sin = _tables(T, n)
    t, i = (sets[0] if T else None), sets[-1]
    out = int8_qkv(t and t["x"], i["x"], heads=heads, weights=(t and t["w"], i["w"]), biases=(t and t["b"], i["b"]),
                   norms=((t and t["q"], i["q"]), (t and t["k"], i["k"])), cos=cos, sin=sin)
    for at in (slice(0, 20), slice(n - 300, n - 240), slice(n - 30, n)):  # (of the image rows)
        part = {**i, "x": Int8Rows(i["x"].q[:, at].contiguous(), i["x"].scale[:, at].contiguous(), K, BF16)}
        place = slice(T + at.start, T + at.stop)
        _check_qkv(out[:, :, place], [part], heads, cos[place], sin[place])
    if T:
        _check_qkv(out[:, :, :T], [t], heads, cos[:T], sin[:T])


def test_qkv_parts_may_be_missing():
    gen = _gen(8)
    B, n, heads, K = 2, 70, 2, 192
    s = _qkv_set(gen, B, n, K, heads, BF16, bias=False, norms=False)
    out = int8_qkv(None, s["x"], heads=heads, weights=(None, s["w"]))
    _check_qkv(out, [s], heads, None, None)
    cos, sin = _tables(0, n)
    _check_qkv(int8_qkv(None, s["x"], heads=heads, weights=(None, s["w"]), cos=cos, sin=sin), [s], heads, cos, sin)
    # tables whose pairs differ, as no pair of rotary tables does but the call allows
    cos, sin = torch.rand(n, 128, device="cuda", generator=gen), torch.rand(n, 128, device="cuda", generator=gen)
    _check_qkv(int8_qkv(None, s["x"], heads=heads, weights=(None, s["w"]), cos=cos, sin=sin), [s], heads, cos, sin)


def test_qkv_into_a_view_and_from_16_bit_rows():
    gen = _gen(9)
    B, T, n, heads, K = 2, 6, 40, 3, 200
    text, image = _randn(gen, B, T, K), _randn(gen, B, n, K)
    ws = [quantize_weight(_randn(gen, 3 * heads * 128, K, std=0.05)) for _ in range(2)]
    want = int8_qkv(quantize_rows(text), quantize_rows(image), heads=heads, weights=ws)
    buf = torch.full((3, B, T + n + 4, heads + 1, 128), 5.0, dtype=BF16, device="cuda")
    view = buf[:, :, 2:2 + T + n, :heads]
    assert int8_qkv(text, image, heads=heads, weights=ws, out=view) is view
    assert torch.equal(view, want)
    view.fill_(5.0)
    assert (buf == 5).all()
    # an empty text is no text
    cos, sin = _tables(0, n)
    a = int8_qkv(text[:, :0], image, heads=heads, weights=ws, cos=cos, sin=sin)
    assert torch.equal(a, int8_qkv(None, image, heads=heads, weights=(None, ws[1]), cos=cos, sin=sin))


def test_qkv_keeps_bad_rows_to_themselves():
    gen = _gen(10)
    x = _randn(gen, 1, 40, 128)
    x[0, 7, 3] = float("nan")
    w = _weight(gen, 3 * 2 * 128, 128)
    out = int8_qkv(None, x, heads=2, weights=(None, w))
    assert torch.isnan(out[:, 0, 7]).all()
    keep = [i for i in range(40) if i != 7]
    assert torch.isfinite(out[:, 0, keep]).all()


# ------------------------------------------------------------------ sizes past 32 bits
def _free(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


def test_outputs_past_31_bits():
    _free(16)
    gen = _gen(21)
    M, N, K = 280000, 8200, 64
    x, w = _rows(gen, M, K), _weight(gen, N, K)
    out = int8_linear(x, w)
    for at in (slice(0, 3), slice(M - 3, M), slice(M // 2, M // 2 + 3)):
        _check_linear(out[at], Int8Rows(x.q[at], x.scale[at], K, BF16), w, None)


def test_rows_past_31_bits():
    _free(24)
    gen = _gen(22)
    M, K, N = 40000, 1 << 16, 40
    x = torch.zeros(M, K, dtype=BF16, device="cuda")
    last = _randn(gen, 5, K)
    x[-5:] = last
    r = quantize_rows(x)
    assert torch.equal(r.q[-5:].long(), O.quantize(last)[0]) and not r.q[:-5].any()
    w = _weight(gen, N, K)
    out = int8_linear(r, w)
    _check_linear(out[-5:], Int8Rows(r.q[-5:], r.scale[-5:], K, BF16), w, None)
    assert not out[:-5].any()


# ------------------------------------------------------------------ streams, graphs, together
def _chain(s):
    """A double block's way from its residual stream through Q/K/V and one linear layer back to it."""
    rows, text = adaln_quantize_pair(dict(x=s["x"], shift=s["sh"], scale=s["sc"], y=s["y"], gate=s["g"], x_out=s["xo"]),
                                     dict(x=s["c"], shift=s["sh"], scale=s["sc"]))
    qkv = int8_qkv(text, rows, heads=s["heads"], weights=s["w"], norms=s["norms"], cos=s["cos"], sin=s["sin"])
    o = qkv[2].flatten(2)  # V stands in for attention
    return rows, text, qkv, int8_linear(quantize_rows(o), s["wo"], s["bo"], gelu=True)


def _chain_state(seed, heads=2, T=8, n=100):
    gen = _gen(seed)
    C = heads * 128
    mod = _randn(gen, 2, 3 * C, std=0.3)
    sh, sc, g = mod.chunk(3, 1)
    x = _randn(gen, 2, n, C)
    return dict(x=x, y=_randn(gen, 2, n, C), xo=torch.empty_like(x), c=_randn(gen, 2, T, C), sh=sh, sc=sc, g=g, heads=heads,
                w=(_weight(gen, 3 * C, C), _weight(gen, 3 * C, C)), wo=_weight(gen, 300, C), bo=_randn(gen, 300),
                norms=tuple((_randn(gen, 128), _randn(gen, 128)) for _ in range(2)), **dict(zip(("cos", "sin"), _tables(T, n))))


def _check_chain(s, rows, text, qkv, out):
    _check_adaln(rows, s["x"], s["sh"], s["sc"], s["y"], s["g"], s["xo"])
    _check_adaln(text, s["c"], s["sh"], s["sc"])
    sets = [dict(x=r, w=w, b=None, q=q, k=k) for r, w, q, k in zip((text, rows), s["w"], *s["norms"])]
    _check_qkv(qkv, sets, s["heads"], s["cos"], s["sin"])
    o = quantize_rows(qkv[2].flatten(2))
    _check_linear(out, o, s["wo"], s["bo"], True)


def test_a_block_runs_together():
    s = _chain_state(31)
    _check_chain(s, *_chain(s))


def test_another_stream():
    s = _chain_state(32)
    want = _chain(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _chain(s)
    side.synchronize()
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])


def test_graph_replays():
    s = _chain_state(33)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _chain(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _chain(s)
    for seed in range(3):
        gen = _gen(seed)
        for k in ("x", "y", "c"):
            s[k].copy_(_randn(gen, *s[k].shape))
        graph.replay()
        torch.cuda.synchronize()
        residual = s["xo"].clone()
        _check_chain(s, *got)
        want = _chain(s)  # eager work between the replays
        for a, b in zip((got[0].q, got[1].q, got[2], got[3], residual), (want[0].q, want[1].q, want[2], want[3], s["xo"])):
            assert torch.equal(a, b)


def test_two_launches_in_a_graph():
    """A product whose last rows go apart, captured and replayed among eager calls on new rows."""
    gen = _gen(31)
    M, N, K = 16819, 3064, 1400
    w, b = _weight(gen, N, K), _randn(gen, N)
    x = _rows(gen, M, K)
    out = torch.empty(M, N, dtype=BF16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        int8_linear(x, w, b, gelu=True, out=out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            int8_linear(x, w, b, gelu=True, out=out)
        for _ in range(3):
            q, scale = _int8(gen, M, K)
            x.q.copy_(q)
            x.scale.copy_(scale)
            out.zero_()
            graph.replay()
            want = int8_linear(x, w, b, gelu=True)
            stream.synchronize()
            assert torch.equal(out, want)


def test_the_same_twice():
    s = _chain_state(34)
    a, b = _chain(s), _chain(s)
    assert torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])


def test_operators_are_traceable():
    s = _chain_state(35)
    x, w = quantize_rows(s["x"]), s["wo"]
    out = torch.empty(2, 100, 300, dtype=BF16, device="cuda")
    hip, checks = torch.ops.hilberta_hip, ("test_schema", "test_faketensor")
    for op, args in ((hip.int8_rows, (s["x"],)), (hip.int8_linear, (x.q, x.scale, w.q, w.scale, s["bo"], BF16, True)),
                     (hip.int8_linear_rows, (s["x"], w.q, w.scale, None, False)),
                     (hip.int8_linear_out, (x.q, x.scale, w.q, w.scale, s["bo"], out, True)),
                     (hip.int8_adaln, (s["x"], s["sh"], s["sc"], s["y"], s["g"], s["xo"], 1e-6)),
                     (hip.int8_adaln_pair, (s["x"], s["sh"], s["sc"], s["y"], s["g"], s["xo"],
                                            s["c"], s["sh"], s["sc"], None, None, None, 1e-6))):
        torch.library.opcheck(op.default, args, test_utils=checks)
    t, (wt, wi), ((qt, qi), (kt, ki)) = quantize_rows(s["c"]), s["w"], s["norms"]
    sets = (t.q, t.scale, wt.q, wt.scale, None, qt, kt, x.q, x.scale, wi.q, wi.scale, None, qi, ki, s["cos"], s["sin"])
    qkv = torch.empty(3, 2, s["cos"].shape[0], s["heads"], 128, dtype=BF16, device="cuda")
    torch.library.opcheck(hip.int8_qkv.default, (*sets, BF16, s["heads"], 1e-6), test_utils=checks)
    torch.library.opcheck(hip.int8_qkv_out.default, (*sets, qkv, 1e-6), test_utils=checks)
    torch.library.opcheck(hip.int8_linear_rows.default, (s["x"][:1, :3], w.q, w.scale, s["bo"], True), test_utils=checks)
    assert torch.equal(hip.int8_qkv.default(*sets, BF16, s["heads"], 1e-6), hip.int8_qkv_out.default(*sets, qkv, 1e-6) or qkv)


def test_gradients_are_refused():
    s = _chain_state(37)
    w, b = s["wo"], s["bo"].clone().requires_grad_()
    for call in (lambda: int8_linear(s["x"][:1, :3], w, b), lambda: int8_linear(s["x"], w, b),
                 lambda: quantize_rows(s["x"].clone().requires_grad_()),
                 lambda: int8_linear(s["x"], w, out=torch.empty(2, 100, 300, dtype=BF16, device="cuda", requires_grad=True))):
        with pytest.raises(ValueError, match="Inference only"):
            call()
    with torch.no_grad():
        assert torch.equal(int8_linear(s["x"], w, b), int8_linear(s["x"], w, b.detach()))
    with torch.inference_mode():
        assert int8_linear(s["x"], w, b).shape == (2, 100, 300)


def test_writes_count_for_autograd():
    """A tensor saved for a backward and then written here fails that backward."""
    s = _chain_state(36)
    p = torch.ones(2, 100, 300, dtype=BF16, device="cuda", requires_grad=True)
    buf = torch.zeros(2, 100, 300, dtype=BF16, device="cuda")
    z = (p * buf).sum()
    int8_linear(quantize_rows(s["x"]), s["wo"], out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
