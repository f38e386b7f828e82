"""flux_norm.group_norm on the GPU against its definition in 64 bits (oracle/layer_ops.py): both kinds of launches, all types,
odd sizes, layouts, in place, streams and graphs."""

import pytest
import torch

from hilberta_amd.flux_linear import linear
from hilberta_amd.flux_norm import group_norm
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
BF16, HALF, FLOAT = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, HALF, FLOAT]


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


def _normal(*shape, dtype=BF16, std=1.0, mean=0.0, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed + sum(shape))
    return (mean + std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


def _rows(B, P, C, dtype=BF16, seed=0):
    """Channels with means and sizes of their own."""
    x = _normal(B, P, C, dtype=FLOAT, seed=seed)
    return (x * (0.5 + torch.rand(C, device="cuda")) + 2 * _normal(C, dtype=FLOAT, seed=seed + 1)).to(dtype)


def _check(got, x, groups, weight=None, bias=None, act=None, eps=1e-6):
    exact, bound = L.group_norm(x, groups, weight, bias, act, eps)
    assert got.shape == exact.shape and got.dtype == x.dtype
    ok = L.held(got, exact, bound)
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} values off, first at {(~ok).nonzero()[0].tolist()}"
    # (so many additions are nowhere near their bound: all together the values are off by less than a rounding each, and
    # fp32's by the statistics' few)
    assert L.relative(got, exact) <= (torch.finfo(x.dtype).eps / 2 if x.dtype != FLOAT else 1e-6)


# (batch, pixels, channels, groups): groups that fit a workgroup, and chunks; one channel a group, one group, odd counts
SIZES = [
    (1, 1, 1, 1), (1, 1, 64, 32), (3, 1, 60, 12), (2, 7, 5, 5), (1, 100, 512, 32), (2, 256, 512, 32), (3, 1961, 60, 12), (1, 300, 9, 3),
    (2, 64, 96, 6), (5, 33, 320, 32), (1, 1024, 640, 32), (1, 2048, 1, 1), (1, 2049, 1, 1), (1, 3000, 8, 1), (1, 4096, 512, 32),
    (2, 5000, 128, 32), (1, 16384, 512, 32), (1, 10007, 60, 12), (2, 9000, 20, 4), (1, 4100, 2560, 32), (1, 700, 8192, 32), (1, 600, 8190, 2),
    (1, 65536, 128, 32), (1, 70001, 24, 8), (3, 40000, 7, 7), (1, 5000, 256, 256), (1, 3000, 1000, 1), (600, 40, 64, 2), (1, 300000, 16, 16),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, P, C, G", SIZES)
def test_sizes(B, P, C, G, dtype):
    x, w, b = _rows(B, P, C, dtype), _normal(C, dtype=dtype, mean=1.0, std=0.1), _normal(C, dtype=dtype, std=0.1)
    _check(group_norm(x, G, w, b), x, G, w, b)
    _check(group_norm(x, G, w, b, act="silu"), x, G, w, b, "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P", [64, 20000])
def test_without_weights_and_other_eps(P, dtype):
    x, w = _rows(2, P, 64, dtype), _normal(64, dtype=dtype)
    _check(group_norm(x, 8), x, 8)
    _check(group_norm(x, 8, w, eps=0.1), x, 8, w, eps=0.1)
    _check(group_norm(x, 8, None, w, act="silu", eps=1e-5), x, 8, None, w, "silu", 1e-5)


@pytest.mark.parametrize("P, C, G", [(100, 64, 8), (5000, 64, 8), (90000, 128, 32)])
def test_means_far_from_zero(P, C, G):
    """A deviation of 1 about 1000, and 1 about 1e4 in some channels' groups: the mean's own rounding is 6e-5 of it."""
    x = _normal(1, P, C, dtype=FLOAT, mean=1000.0)
    got, (exact, bound) = group_norm(x, G), L.group_norm(x, G)
    assert L.held(got, exact, bound).all() and L.relative(got, exact) < 2e-4
    x[..., :C // 2] += 9000
    got, (exact, bound) = group_norm(x, G), L.group_norm(x, G)
    assert L.held(got, exact, bound).all() and L.relative(got, exact) < 2e-3


@pytest.mark.parametrize("P", [50, 9000])
def test_constant_groups_and_outliers(P):
    x = _normal(1, P, 32, dtype=FLOAT)
    x[..., :8] = 3.25            # no deviation: exactly the bias
    x[:, 0, 8:16] = 1e6          # (the first pixel far from the others)
    b = _normal(32, dtype=FLOAT)
    got, (exact, bound) = group_norm(x, 4, None, b), L.group_norm(x, 4, None, b)
    assert torch.equal(got[..., :8], b[:8].expand(1, P, 8))
    assert L.held(got, exact, bound).all() and L.relative(got[..., 8:16], exact[..., 8:16]) < 1e-5


def test_a_dark_half():
    """Chunks whose means differ by far more than the deviation within them."""
    x = _normal(1, 100000, 64, dtype=FLOAT, std=1e-2)
    x[:, 60000:] += 100
    x[:, :300] -= 1000
    got, (exact, bound) = group_norm(x, 8), L.group_norm(x, 8)
    assert L.held(got, exact, bound).all() and L.relative(got, exact) < 2e-6


@pytest.mark.parametrize("P", [50, 9000])
def test_infinities_and_nans_stay_in_their_groups(P):
    x = _normal(2, P, 64)
    clean = group_norm(x, 8, act="silu")
    x[0, 3, 9], x[1, P - 1, 63] = float("nan"), float("inf")
    got = group_norm(x, 8, act="silu")
    assert got[0, :, 8:16].isnan().all() and got[1, :, 56:].isnan().any()
    got[0, :, 8:16], got[1, :, 56:] = clean[0, :, 8:16], clean[1, :, 56:]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(6, 5), (80, 110)])
def test_images(size, dtype):
    """Channels-last images and videos, column blocks and row ranges, in place; torch's own order of dimensions comes back."""
    x = _rows(2, size[0] * size[1], 48, dtype)
    want = group_norm(x, 6, act="silu")
    image = x.unflatten(1, size).permute(0, 3, 1, 2)
    got = group_norm(image, 6, act="silu")
    assert got.shape == image.shape and got.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(got.permute(0, 2, 3, 1).flatten(1, 2), want)
    video = x.unflatten(1, (2, size[0] // 2, size[1])).permute(0, 4, 1, 2, 3)
    got = group_norm(video, 6, act="silu")
    assert got.is_contiguous(memory_format=torch.channels_last_3d) and torch.equal(got.permute(0, 2, 3, 4, 1).flatten(1, 3), want)
    for shift in (1, 2, 8):
        wide = _normal(3, size[0] * size[1] + 2, 48 + shift + 3, dtype=dtype)
        wide[:2, 1:-1, shift:shift + 48] = x
        part, before = wide[:2, 1:-1, shift:shift + 48], wide.clone()
        assert torch.equal(group_norm(part, 6, act="silu"), want)
        version = wide._version
        assert group_norm(part, 6, act="silu", out=part) is part and wide._version > version
        assert torch.equal(part, want)
        part.copy_(x)
        assert torch.equal(wide, before)
    one = x[:, :1].expand(2, 40, 48)  # (pixels that repeat)
    assert torch.equal(group_norm(one, 6), group_norm(one.contiguous(), 6))
    one = x[:1].expand(3, -1, 48)
    assert torch.equal(group_norm(one, 6, act="silu"), want[:1].expand(3, -1, 48))


def test_nothing_to_do():
    assert group_norm(_normal(0, 5, 8), 2).shape == (0, 5, 8)
    assert group_norm(_normal(2, 0, 8), 2).shape == (2, 0, 8)
    assert group_norm(_normal(2, 0, 3, 8).permute(0, 3, 1, 2), 2).shape == (2, 8, 0, 3)


def test_same_results_again_and_on_another_stream():
    for P in (60, 30000):
        x = _normal(2, P, 128)
        want = group_norm(x, 32, act="silu")
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [group_norm(x, 32, act="silu") for _ in range(4)]
        stream.synchronize()
        assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("P", [64, 5000, 40000])
def test_graph_replays(P):
    x, y, w = _normal(1, P, 128), torch.empty(1, P, 128, dtype=BF16, device="cuda"), _normal(128)
    group_norm(x, 32, w, act="silu", out=y)  # (warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = group_norm(x, 32, w, act="silu")
        group_norm(z, 16, out=y)
    for seed in range(3):
        x.copy_(_normal(1, P, 128, seed=seed + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, group_norm(x, 32, w, act="silu")) and torch.equal(y, group_norm(z, 16))
        group_norm(_normal(2, 3000, 256), 32)
        torch.cuda.synchronize()


def test_operators():
    hip = torch.ops.hilberta_hip
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    x, w = _normal(2, 6, 5, 16).permute(0, 3, 1, 2), _normal(16)
    torch.library.opcheck(hip.group_norm.default, (x, 4, w, w, True, 1e-6), test_utils=checks)
    torch.library.opcheck(hip.group_norm.default, (_normal(2, 30, 16), 4, None, None, False, 1e-6), test_utils=checks)
    torch.library.opcheck(hip.group_norm_out.default, (x, 4, w, None, torch.empty_like(x), True, 1e-6), test_utils=checks)


def test_with_the_linear_layers():
    """A decoder's middle attention as it would be run: norm, Q/K/V of the pixels, attention, output with the residual; and a
    residual block's shortcut of one-pixel convolutions."""
    B, P, C = 2, 240, 128
    x, gw, gb = _rows(B, P, C), _normal(C, mean=1.0, std=0.1), _normal(C, std=0.1)
    wq, bq = _normal(3 * C, C, std=C**-0.5), _normal(3 * C, std=0.02)
    wo, bo = _normal(C, C, std=C**-0.5, seed=3), _normal(C, std=0.02, seed=3)
    ws, bs = _normal(2 * C, C, std=C**-0.5, seed=5), _normal(2 * C, std=0.02, seed=5)
    h = group_norm(x, 32, gw, gb)
    qkv = linear(h, wq, bq)
    q, k, v = qkv.float().chunk(3, -1)
    a = (torch.softmax(q @ k.transpose(1, 2).contiguous() * C**-0.5, -1) @ v).to(BF16)
    stream = x.clone()
    linear(a, wo, bo, residual=stream, out=stream)
    body = linear(group_norm(stream, 32, gw, gb, act="silu"), ws, bs, act="silu")
    out = linear(stream, ws, bs, residual=body)
    # each step in 64 bits from what the step before returned
    _check(h, x, 32, gw, gb)
    steps = [(qkv, dict(x=h, weight=wq, bias=bq)), (stream, dict(x=a, weight=wo, bias=bo, residual=x)),
             (body, dict(x=group_norm(stream, 32, gw, gb, act="silu"), weight=ws, bias=bs, act="silu")),
             (out, dict(x=stream, weight=ws, bias=bs, residual=body))]
    for got, args in steps:
        exact, bound = L.linear(**args)
        assert L.held(got, exact, bound).all()
    # and the whole of it, whose few 16-bit roundings add up to no more than 8 steps of its size
    f8 = lambda t: t.double()  # noqa: E731
    h8 = L.group_norm(x, 32, gw, gb)[0]
    q, k, v = (h8 @ f8(wq).T + f8(bq)).chunk(3, -1)
    s8 = f8(x) + torch.softmax(q @ k.transpose(1, 2).contiguous() * C**-0.5, -1) @ v @ f8(wo).T + f8(bo)
    b8 = L.activate(L.group_norm(s8, 32, gw, gb, "silu")[0] @ f8(ws).T + f8(bs), "silu")
    o8 = s8 @ f8(ws).T + f8(bs) + b8
    assert L.relative(out, o8) < 8 * torch.finfo(BF16).eps / 2
