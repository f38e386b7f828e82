"""flux_linear and flux_norm.group_norm on tensors of more than 2^31 elements, whose last offsets pass 32 bits."""

import pytest
import torch

from hilberta_amd.flux_linear import linear
from hilberta_amd.flux_norm import group_norm
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROWS, WIDTH = 262145, 8200  # 2.15e9 elements


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    yield
    torch.cuda.empty_cache()


def _normal(*shape, std=1.0):
    gen = torch.Generator("cuda").manual_seed(sum(shape))
    return torch.empty(shape, dtype=BF16, device="cuda").normal_(0, std, generator=gen)


def _check(got, act=None, **args):
    exact, bound = L.linear(act=act, **args)
    assert L.held(got, exact, bound).all() and L.relative(got, exact) <= torch.finfo(got.dtype).eps / 2


SAMPLES = [slice(0, 300), slice(131000, 131300), slice(261880, 262145)]  # (2^31 elements end in row 261887)


@pytest.mark.parametrize("K", [64, 1024])
def test_outputs_and_residual(K):
    x, w, b, gate = _normal(ROWS, K), _normal(WIDTH, K, std=K**-0.5), _normal(WIDTH), _normal(1, WIDTH)
    res = _normal(ROWS, WIDTH)
    want = [res[s].clone() for s in SAMPLES]
    assert linear(x, w, b, residual=res, gate=gate, out=res) is res
    for s, before in zip(SAMPLES, want):
        _check(res[s], x=x[s], weight=w, bias=b, residual=before, gate=gate)


@pytest.mark.parametrize("columns", [slice(100, 164), slice(101, 166), slice(8000, 8200)])
def test_rows_far_apart(columns):
    """A column block of a wider buffer as rows, in direct loads and by registers."""
    x = _normal(ROWS, WIDTH)[:, columns]
    w = _normal(72, x.shape[1], std=0.1)
    got = linear(x, w, act="silu")
    for s in SAMPLES:
        _check(got[s], x=x[s], weight=w, act="silu")


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("odd", [0, 1])
def test_weights(rows, odd):
    """Every kind of kernel: a few rows, tiles, and weights of an odd length that are copied or go by registers."""
    w = _normal(ROWS, WIDTH + odd, std=WIDTH**-0.5)
    x = _normal(rows, WIDTH + odd)
    got = linear(x, w)
    for s in SAMPLES:
        _check(got[:, s], x=x, weight=w[s])


def test_an_image():
    """One image of 2^31 + 24 values; at most 1024 pixels a thread in eights, 38 additions in a workgroup and 10 joins."""
    P, C, G = (1 << 28) + 3, 8, 2
    x, w, b = _normal(1, P, C), _normal(C), _normal(C)
    x[:, : P // 3] += 2
    parts = [slice(i, min(i + (1 << 24), P)) for i in range(0, P, 1 << 24)]
    n = P * C // G
    mean = sum(x[0, s].double().unflatten(1, (G, -1)).sum((0, 2)) for s in parts) / n
    var = sum((x[0, s].double().unflatten(1, (G, -1)) - mean[:, None]).square().sum((0, 2)) for s in parts) / n
    statistics = mean.view(1, 1, G, 1), var.view(1, 1, G, 1)
    got = group_norm(x, G, w, b, act="silu")
    for s in parts:
        exact, bound = L.group_norm(x[:, s], G, w, b, "silu", steps=200, statistics=statistics)
        assert L.held(got[:, s], exact, bound).all()
        assert L.relative(got[:, s], exact) <= torch.finfo(BF16).eps / 2
    assert group_norm(x, G, w, b, act="silu", out=x) is x
    assert all(torch.equal(x[:, s], got[:, s]) for s in parts)
