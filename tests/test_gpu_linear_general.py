"""The wide kernel's epilogue through LDS (tests/linear_calls.py has the sizes, tests/test_linear_choice.py their route): tiles of
several batch elements, columns that are no multiple of eight, outputs at any element, against the definition in 64 bits."""

import pytest
import torch

from hilberta_amd.flux_linear import linear, linear_pair
from oracle import layer_ops as L
from tests.linear_calls import GENERAL, GENERAL_PAIRS, SHIFTS

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


def _normal(*shape, dtype=torch.bfloat16, std=1.0, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed + sum(shape))
    return (std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


def _set(batch, rows, K, N, more, dtype=torch.bfloat16, bias=True, seed=0):
    s = dict(x=_normal(batch, rows, K, dtype=dtype, seed=seed), weight=_normal(N, K, dtype=dtype, std=K**-0.5, seed=seed + 1),
             bias=_normal(N, dtype=dtype, seed=seed + 2) if bias else None)
    if more:
        s["residual"] = _normal(batch, rows, N, dtype=dtype, seed=seed + 3)
    if more == "gate":
        s["gate"] = _normal(batch, N, dtype=dtype, std=0.5, seed=seed + 4)
    return s


def _check(got, act=None, **args):
    exact, bound = L.linear(act=act, **args)
    assert got.shape == exact.shape and got.dtype == args["x"].dtype
    ok = L.held(got, exact, bound)
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} values off, first at {(~ok).nonzero()[0].tolist()}"
    assert L.relative(got, exact) <= torch.finfo(got.dtype).eps / 2


@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("more", ["", "residual", "gate"])
@pytest.mark.parametrize("size", GENERAL)
def test_epilogues(size, more, act):
    s = _set(*size, more, dtype=torch.float16 if act == "silu" else torch.bfloat16, bias=act != "gelu")
    _check(linear(**s, act=act), act=act, **s)


@pytest.mark.parametrize("shift, longer", SHIFTS)
@pytest.mark.parametrize("more", ["", "residual", "gate"])
@pytest.mark.parametrize("size", GENERAL)
def test_into_a_wider_buffer(size, more, shift, longer):
    """In place where there is a residual; what lies beside the rows stays."""
    batch, rows, _, N = size
    s = _set(*size, more)
    flat = _normal(shift + batch * (rows + 1) * (N + longer), seed=9)
    held = flat[shift:].view(batch, rows + 1, N + longer)
    before, out = held.clone(), held[:, :rows, :N]
    if more:
        s["residual"] = out
    assert linear(**s, out=out) is out
    if more:
        s["residual"] = before[:, :rows, :N]
    _check(out, **s)
    out.copy_(before[:, :rows, :N])
    assert torch.equal(held, before)


@pytest.mark.parametrize("mores", [("", ""), ("gate", "gate"), ("residual", "residual")])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("size", GENERAL_PAIRS)
def test_pairs(size, act, mores):
    batch, rows, K, N = size
    sets = [_set(batch, m, K, N, more, seed=20 * i) for i, (m, more) in enumerate(zip(rows, mores))]
    for out, s in zip(linear_pair(*sets, act=act), sets):
        _check(out, act=act, **s)


@pytest.mark.parametrize("mores", [("", "gate"), ("gate", "residual")])
def test_pairs_whose_sets_differ(mores):
    """Deep enough for the wide kernel, whose one epilogue for both is the general one."""
    sets = [_set(1, m, 1032, 4000, more, seed=20 * i) for i, (m, more) in enumerate(zip((512, 2048), mores))]
    for out, s in zip(linear_pair(*sets), sets):
        _check(out, **s)


def test_rows_stay_apart():
    """Infinities and NaN of one row and one channel, rows of several batch elements in a tile."""
    s = _set(315, 13, 776, 4089, "gate")
    clean = linear(**s)
    s["x"][3, 5, 7], s["x"][200, 12, 775] = float("inf"), float("nan")
    s["weight"][4088, 0] = s["gate"][77, 100] = float("nan")
    got = linear(**s)
    assert not got[3, 5].isfinite().any() and got[200, 12].isnan().all() and got[..., 4088].isnan().all() and got[77, :, 100].isnan().all()
    for t in (got, clean):
        t[3, 5] = t[200, 12] = t[..., 4088] = t[77, :, 100] = 0
    assert torch.equal(got, clean)
