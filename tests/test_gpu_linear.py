"""flux_linear on the GPU against its definition in 64 bits (oracle/layer_ops.py): every kernel and epilogue, both types, odd
sizes, rows at any address, row ranges and column blocks, in place, two row sets, streams and graphs."""

import pytest
import torch

from hilberta_amd.flux_linear import linear, linear_pair
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
BF16, HALF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


def _normal(*shape, dtype=BF16, std=1.0, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed + sum(shape))
    return (std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


def _layer(K, N, dtype=BF16, bias=True, seed=0):
    return dict(weight=_normal(N, K, dtype=dtype, std=K**-0.5, seed=seed + 1), bias=_normal(N, dtype=dtype, seed=seed + 2) if bias else None)


def _check(got, act=None, **args):
    exact, bound = L.linear(act=act, **args)
    assert got.shape == exact.shape and got.dtype == args["x"].dtype
    ok = L.held(got, exact, bound)
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} values off, first at {(~ok).nonzero()[0].tolist()}"
    # (so many additions are nowhere near their bound: all together the values are off by less than a rounding each)
    assert L.relative(got, exact) <= torch.finfo(got.dtype).eps / 2


# (rows in all, features, columns): a few rows; each of the smaller tiles; the wide kernel at edges
SIZES = [
    (1, 1, 1), (1, 8, 16), (1, 7, 5), (3, 127, 33), (5, 129, 16), (16, 1024, 100), (16, 3, 1000), (1, 5000, 24), (2, 100, 4097),
    (17, 1, 1), (17, 64, 32), (33, 65, 31), (100, 200, 64), (40, 1000, 3000), (77, 320, 1000), (130, 72, 129), (256, 512, 96),
    (500, 136, 1500), (640, 640, 640), (1000, 1000, 1001), (1025, 64, 2049), (300, 4096, 300), (512, 2048, 96),
    (2048, 640, 2048), (1000, 1096, 4001), (4096, 64, 2048), (4095, 72, 4097), (5000, 8, 4000), (4096, 1024, 4096), (2500, 130, 8000),
]


@pytest.mark.parametrize("dtype", [BF16, HALF])
@pytest.mark.parametrize("rows, K, N", SIZES)
def test_sizes(rows, K, N, dtype):
    x, layer = _normal(rows, K, dtype=dtype), _layer(K, N, dtype)
    _check(linear(x, **layer), x=x, **layer)


EPILOGUES = [(act, bias, more) for act in (None, "gelu", "silu") for bias in (True, False) for more in ("", "residual", "gate")]


# rows that are no multiple of 16 bytes: copied first, where that pays, or not
@pytest.mark.parametrize("dtype", [BF16, HALF])
@pytest.mark.parametrize("rows, K, N", [(17, 3, 40), (17, 9, 16), (20, 13, 2405), (65, 63, 65), (64, 57, 64), (130, 58, 129), (300, 71, 1000), (999, 1001, 777),
                                        (77, 4097, 3072), (40, 5003, 500), (18, 7001, 33), (2000, 5001, 5000), (600, 2999, 4001)])
def test_rows_of_odd_lengths(rows, K, N, dtype):
    x, layer = _normal(rows, K, dtype=dtype), _layer(K, N, dtype)
    _check(linear(x, **layer), x=x, **layer)
    pair = linear_pair(dict(x=x[None], **layer), dict(x=x[None, 5:17], **layer))
    for got, rows_of in zip(pair, (x, x[5:17])):
        _check(got[0], x=rows_of, **layer)


@pytest.mark.parametrize("act, bias, more", EPILOGUES)
@pytest.mark.parametrize("batch, rows, K, N", [(3, 61, 99, 201), (1, 1, 64, 100), (3, 5, 200, 72), (2, 33, 96, 200), (3, 170, 136, 1000), (2, 2048, 128, 4096),
                                               (3, 1365, 128, 4096), (1, 4173, 128, 4104), (2, 2048, 72, 4008)])
def test_epilogues(batch, rows, K, N, act, bias, more):
    x, layer = _normal(batch, rows, K), _layer(K, N, bias=bias)
    if more:
        layer["residual"] = _normal(batch, rows, N, seed=5)
    if more == "gate":
        layer["gate"] = _normal(batch, N, std=0.5, seed=6)
    _check(linear(x, act=act, **layer), act=act, x=x, **layer)


@pytest.mark.parametrize("act, more", [("gelu", ""), ("silu", ""), (None, "residual"), (None, "gate"), ("gelu", "gate")])
def test_epilogues_in_half_precision(act, more):
    x, layer = _normal(2, 2048, 192, dtype=HALF), _layer(192, 4096, HALF)
    if more:
        layer["residual"] = _normal(2, 2048, 4096, dtype=HALF, seed=5)
    if more == "gate":
        layer["gate"] = _normal(2, 4096, dtype=HALF, std=0.5, seed=6)
    _check(linear(x, act=act, **layer), act=act, x=x, **layer)


def test_long_sums():
    """The deepest of the transformer's layers, where the sums' own error shows if they are not fp32."""
    for rows in (1, 77, 512, 4096):
        x, layer = _normal(rows, 12288), _layer(12288, 3072)
        got = linear(x, **layer)
        exact, _ = L.linear(x, **layer)
        assert L.relative(got, exact) <= torch.finfo(BF16).eps / 2


# few tiles over many features, which several workgroups share
PARTS = [(126, 13952, 27), (383, 5200, 5024), (127, 8104, 5270), (17, 1543, 16), (20, 3001, 100), (100, 12345, 300), (1000, 8192, 520),
         (512, 12288, 3072), (700, 9001, 1500), (1100, 8200, 1001), (513, 6000, 2048),
         (1, 12288, 10), (8, 12288, 512), (16, 14633, 129), (5, 7000, 1024)]


@pytest.mark.parametrize("dtype", [BF16, HALF])
@pytest.mark.parametrize("rows, K, N", PARTS)
def test_features_in_parts(rows, K, N, dtype):
    x, layer = _normal(rows, K, dtype=dtype), _layer(K, N, dtype)
    _check(linear(x, **layer), x=x, **layer)


@pytest.mark.parametrize("batch, rows, K, N", [(3, 23, 4096, 203), (3, 171, 12000, 2001)])
@pytest.mark.parametrize("act, bias, more", EPILOGUES)
def test_epilogues_of_parts(batch, rows, K, N, act, bias, more):
    x, layer = _normal(batch, rows, K), _layer(K, N, bias=bias)
    if more:
        layer["residual"] = _normal(batch, rows, N, seed=5)
    if more == "gate":
        layer["gate"] = _normal(batch, N, std=0.5, seed=6)
    _check(linear(x, act=act, **layer), act=act, x=x, **layer)


@pytest.mark.parametrize("text, image, K, N", [(1, 30, 6000, 200), (30, 1, 6000, 200), (77, 100, 6000, 200), (0, 40, 6000, 200),
                                               (77, 256, 12288, 2048), (300, 33, 9999, 1999)])
def test_pairs_in_parts(text, image, K, N):
    sets = []
    for i, rows in enumerate((text, image)):
        s = dict(x=_normal(2, rows, K, seed=i), **_layer(K, N, seed=10 * i))
        if i:
            s |= dict(residual=_normal(2, rows, N, seed=31), gate=_normal(2, N, seed=41))
        sets.append(s)
    for out, s in zip(linear_pair(*sets), sets):
        if s["x"].numel():
            _check(out, **s)


def test_parts_into_a_wider_buffer_and_in_place():
    x, layer, gate = _normal(2, 40, 8000), _layer(8000, 93), _normal(2, 93, seed=3)
    held = _normal(2, 44, 200, seed=9)
    before = held.clone()
    out = held[:, 2:42, 11:104]
    linear(x, **layer, residual=out, gate=gate, out=out)
    _check(out, x=x, **layer, residual=before[:, 2:42, 11:104], gate=gate)
    out.copy_(before[:, 2:42, 11:104])
    assert torch.equal(held, before)


def test_parts_on_two_streams_and_in_a_graph():
    """Calls in flight together have workspaces of their own, and one input's are the same again."""
    x, layer = [_normal(60, 9000, seed=i) for i in range(4)], _layer(9000, 100)
    want = [linear(v, **layer) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = linear(x[i], **layer)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, held = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(linear(x[i], **layer))
        graphs.append(graph)
    for _ in range(3):
        for i in range(2):
            x[i].copy_(_normal(60, 9000, seed=i))
        for h in held:
            h.zero_()
        for g in graphs:
            g.replay()
        linear(x[2], **layer)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("rows", [1, 9, 40, 600, 4096])
def test_rows_anywhere(rows):
    """Row ranges, column blocks at odd columns, transposed batches, expanded rows, views of weights; what lies beside
    the output stays."""
    K, N, batch = 136, 520, 2
    for shift, step in ((0, 0), (8, 0), (3, 0), (0, 5), (1, 8)):
        big = _normal(batch, rows + 3, K + shift + step)
        x = big[:, 2:2 + rows, shift:shift + K]
        weight = _normal(N, K + step, std=K**-0.5)[:, step:]
        bias, gate = _normal(2 * N + 1)[1:1 + N], _normal(batch, 3 * N)[:, N + step:2 * N + step]
        held = _normal(batch, rows + 2, N + shift + step + 2, seed=9)
        before, residual = held.clone(), _normal(batch, rows, N + 1, seed=8)[..., 1:]
        out = held[:, 1:1 + rows, shift:shift + N]
        assert linear(x, weight, bias, residual=residual, gate=gate, out=out) is out
        _check(out, x=x, weight=weight, bias=bias, residual=residual, gate=gate)
        out.copy_(before[:, 1:1 + rows, shift:shift + N])
        assert torch.equal(held, before)
    layer = _layer(K, N)
    x = _normal(rows, batch, K).transpose(0, 1)
    _check(linear(x, **layer), x=x, **layer)
    x = _normal(1, rows, K).expand(batch, rows, K)
    _check(linear(x, **layer), x=x, **layer)
    x = _normal(batch, 1, K).expand(batch, rows, K)
    _check(linear(x, **layer), x=x, **layer)
    _check(linear(x[0], **layer), x=x[0], **layer)


@pytest.mark.parametrize("more", ["", "residual", "gate"])
@pytest.mark.parametrize("rows, N", [(4173, 4104), (4096, 4008), (4351, 4096), (4097, 4096)])
def test_what_lies_beside_tiles_that_are_not_whole_stays(rows, N, more):
    x, layer = _normal(1, rows, 128), _layer(128, N)
    held = _normal(1, rows + 256, N + 264, seed=9)
    before = held.clone()
    out = held[:, 8:8 + rows, 8:8 + N]
    if more:
        layer["residual"] = out
    if more == "gate":
        layer["gate"] = _normal(1, N, std=0.5, seed=6)
    linear(x, **layer, out=out)
    if more:
        layer["residual"] = before[:, 8:8 + rows, 8:8 + N]
    _check(out, x=x, **layer)
    out.copy_(before[:, 8:8 + rows, 8:8 + N])
    assert torch.equal(held, before)


@pytest.mark.parametrize("rows", [1, 60, 700, 4096])
def test_in_place(rows):
    x, layer, stream = _normal(1, rows, 264), _layer(264, 1024), _normal(1, rows, 1024, seed=4)
    gate, before = _normal(1, 1024, seed=3), stream.clone()
    version = stream._version
    assert linear(x, **layer, residual=stream, gate=gate, out=stream) is stream and stream._version > version
    _check(stream, x=x, **layer, residual=before, gate=gate)


@pytest.mark.parametrize("text, image, K, N", [(1, 3, 64, 100), (16, 16, 72, 40), (5, 300, 200, 520), (512, 1024, 256, 768), (77, 4096, 136, 4096),
                                               (256, 4096, 128, 4096), (0, 9, 64, 24), (9, 0, 64, 24), (0, 0, 64, 24)])
@pytest.mark.parametrize("more", ["", "gate", "mixed"])
def test_pairs(text, image, K, N, more):
    sets, act = [], "gelu" if more == "" else None
    for i, rows in enumerate((text, image)):
        s = dict(x=_normal(2, rows, K, seed=i), **_layer(K, N, seed=10 * i))
        if more == "gate" or (more == "mixed" and i):
            s |= dict(residual=_normal(2, rows, N, seed=30 + i), gate=_normal(2, N, seed=40 + i))
        sets.append(s)
    got = linear_pair(*sets, act=act)
    for out, s in zip(got, sets):
        if s["x"].numel():
            _check(out, act=act, **s)
        else:
            assert out.shape == (2, 0, N)


@pytest.mark.parametrize("text, image, K, N", [(77, 4096, 128, 4104), (4173, 300, 72, 4096), (512, 8192, 64, 3000)])
@pytest.mark.parametrize("more", ["", "gate"])
def test_pairs_of_one_element(text, image, K, N, more):
    sets = []
    for i, rows in enumerate((text, image)):
        s = dict(x=_normal(1, rows, K, seed=i), **_layer(K, N, seed=10 * i))
        if more:
            s |= dict(residual=_normal(1, rows, N, seed=30 + i), gate=_normal(1, N, seed=40 + i))
        sets.append(s)
    for out, s in zip(linear_pair(*sets), sets):
        _check(out, **s)


def test_pairs_into_one_buffer():
    both, layer = _normal(1, 1100, 512), [_layer(128, 512, seed=i) for i in (0, 7)]
    x = _normal(1, 1100, 128, seed=3)
    linear_pair(dict(x=x[:, :77], **layer[0], out=both[:, :77]), dict(x=x[:, 77:], **layer[1], out=both[:, 77:]))
    _check(both[:, :77], x=x[:, :77], **layer[0])
    _check(both[:, 77:], x=x[:, 77:], **layer[1])
    both.zero_()  # (one output given, one made)
    made, given = linear_pair(dict(x=x[:, :77], **layer[0]), dict(x=x[:, 77:], **layer[1], out=both[:, 77:]))
    _check(made, x=x[:, :77], **layer[0])
    _check(given, x=x[:, 77:], **layer[1])
    assert given.data_ptr() == both[:, 77:].data_ptr() and not both[:, :77].any()
    given, made = linear_pair(dict(x=x[:, :77], **layer[0], out=both[:, :77]), dict(x=x[:, 77:], **layer[1]))
    _check(given, x=x[:, :77], **layer[0])
    _check(made, x=x[:, 77:], **layer[1])


@pytest.mark.parametrize("rows", [3, 100, 4096])
def test_infinities_and_nans_stay_in_their_rows_and_channels(rows):
    x, layer = _normal(rows, 200), _layer(200, 2000)
    clean = linear(x, **layer)
    x[1, 7], x[2, 199] = float("inf"), float("nan")
    layer["weight"][5, 0] = float("nan")
    got = linear(x, **layer)
    assert got[1, :5].isinf().all() and got[2].isnan().all() and got[:, 5].isnan().all()
    keep_rows = torch.tensor([r for r in range(rows) if r not in (1, 2)], device="cuda")
    keep = torch.tensor([c for c in range(2000) if c != 5], device="cuda")
    assert torch.equal(got[keep_rows][:, keep], clean[keep_rows][:, keep])


def test_what_lies_past_a_row_is_not_read_into_it():
    """NaN in the columns after the rows' and the weight's last feature, and in the rows after them."""
    for rows in (2, 50, 600, 4096):
        for K in (8, 61, 64, 72, 128, 200):
            x, w = _normal(rows + 1, K + 8), _normal(513, K + 8, std=K**-0.5)
            x[:, K:] = w[:, K:] = x[rows:] = w[512:] = float("nan")
            layer = dict(x=x[:rows, :K], weight=w[:512, :K])
            _check(linear(**layer), **layer)


def test_large_values():
    x, w = _normal(64, 128, dtype=HALF) * 60, torch.ones(32, 128, device="cuda", dtype=HALF) * 60
    got, exact = linear(x, w), L.linear(x, w)[0]
    far = exact.abs() > 65536
    assert far.any() and got[far].isinf().all() and torch.equal(got[far].sign().double(), exact[far].sign())
    for act in ("gelu", "silu"):
        v = torch.tensor([[-3e38, -1e4, -90.0, -20.0, -0.0, 0.0, 1e-30, 20.0, 3e38, float("inf")]], device="cuda").to(BF16).T
        got = linear(v, torch.ones(1, 1, device="cuda", dtype=BF16), act=act)[:, 0]
        assert torch.equal(got[6:8], v[6:8, 0] * torch.tensor([0.5, 1.0], device="cuda", dtype=BF16))
        assert got[8].item() == v[8].item() and got[9].isinf() and not got[:7].isnan().any() and (got[:4].abs() < 1e-6).all()


def test_nothing_to_do():
    layer = _layer(64, 40)
    assert linear(_normal(0, 64), **layer).shape == (0, 40)
    assert linear(_normal(2, 0, 64), **layer).shape == (2, 0, 40)
    assert linear(_normal(3, 64), _normal(0, 64)).shape == (3, 0)


def test_same_results_again():
    for rows, K, N in ((1, 3000, 500), (77, 4096, 512), (600, 1000, 777), (4096, 512, 4096)):
        x, layer = _normal(rows, K), _layer(K, N)
        first = linear(x, **layer)
        for _ in range(3):
            assert torch.equal(linear(x, **layer), first)


def test_another_stream():
    x, layer = _normal(700, 333), _layer(333, 999)
    want = linear(x, **layer)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [linear(x, **layer) for _ in range(4)]
    stream.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("rows, K", [(1, 256), (60, 333), (700, 256), (700, 333), (4096, 128)])
def test_graph_replays(rows, K):
    """Captured calls, one with a workspace of its own, replayed among eager ones on other sizes."""
    x, layer, gate = _normal(1, rows, K), _layer(K, 2048), _normal(1, 2048)
    stream = torch.zeros(1, rows, 2048, dtype=BF16, device="cuda")
    linear(x, **layer, residual=stream, gate=gate, out=stream)  # (warm)
    stream.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hidden = linear(x, **layer, act="gelu")
        linear(x, **layer, residual=stream, gate=gate, out=stream)
    for seed in range(3):
        x.copy_(_normal(1, rows, K, seed=seed + 1))
        stream.copy_(_normal(1, rows, 2048, seed=seed))
        before = stream.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(hidden, linear(x, **layer, act="gelu"))
        assert torch.equal(stream, linear(x, **layer, residual=before, gate=gate))
        linear(_normal(90, 777), _normal(80, 777))
        torch.cuda.synchronize()


def test_operators():
    hip = torch.ops.hilberta_hip
    x, layer = _normal(2, 5, 24), _layer(24, 40)
    res, gate = _normal(2, 5, 40), _normal(2, 40)
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    args = (x, layer["weight"], layer["bias"], res, gate)
    torch.library.opcheck(hip.linear.default, (*args, 1), test_utils=checks)
    torch.library.opcheck(hip.linear_out.default, (*args, torch.empty_like(res), 0), test_utils=checks)
    torch.library.opcheck(hip.linear_pair.default, (*args, *args, 2), test_utils=checks)
    torch.library.opcheck(hip.linear_pair_out.default, (*args, torch.empty_like(res), *args, torch.empty_like(res), 2), test_utils=checks)


def test_refusals_on_the_device():
    x, layer = _normal(3, 24), _layer(24, 40)
    with pytest.raises(ValueError, match="one device"):
        linear(x, layer["weight"].cpu())
    with pytest.raises(ValueError, match="Inference only"):
        linear(x, layer["weight"].requires_grad_())
