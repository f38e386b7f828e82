"""The 8-bit operators under torch.func: they record no derivative, so a transform that takes one is refused, with the
reason, before anything else is said about the call."""

import pytest
import torch

from hilberta_amd import flux_int8 as f

BF16 = torch.bfloat16


def _calls(device):
    """Each operator's name: (a call of one of its tensors, that tensor)."""
    zeros = lambda *shape, dtype=BF16: torch.zeros(*shape, dtype=dtype, device=device)  # noqa: E731
    x, v, b = zeros(2, 3, 64), zeros(2, 64), zeros(384)
    rows = f.Int8Rows(zeros(2, 3, 64, dtype=torch.int8), zeros(2, 3, dtype=torch.float32), 64, BF16)
    w = f.Int8Weight(zeros(384, 64, dtype=torch.int8), zeros(384, dtype=torch.float32), 64)
    qkv = lambda b, **out: f.int8_qkv(None, rows, heads=1, weights=(None, w), biases=(None, b), **out)  # noqa: E731
    return {
        "int8_rows": (lambda t: f.quantize_rows(t).scale, x),
        "int8_adaln": (lambda t: f.adaln_quantize(x, t, v).scale, v),
        "int8_adaln with x_out": (lambda t: f.adaln_quantize(x, t, v, y=x, gate=v, x_out=torch.zeros_like(x)).scale, v),
        "int8_adaln_pair": (lambda t: f.adaln_quantize_pair(dict(x=x, shift=v, scale=v), dict(x=x, shift=t, scale=v))[1].scale, v),
        "int8_linear": (lambda t: f.int8_linear(rows, w, t), b),
        "int8_linear of its scales": (lambda t: f.int8_linear(rows._replace(scale=t), w), rows.scale),
        "int8_linear_rows": (lambda t: f.int8_linear(t, w), x),
        "int8_linear_out": (lambda t: f.int8_linear(rows, w, t, out=zeros(2, 3, 384)), b),
        "int8_linear_pair_out": (lambda t: f.int8_linear_pair(dict(x=rows, weight=w), dict(x=rows, weight=w, bias=t))[1], b),
        "int8_qkv": (qkv, b),
        "int8_qkv_out": (lambda t: qkv(t, out=zeros(3, 2, 3, 1, 128)), b),
    }


NAMES = list(_calls("cpu"))


def _refused(name, call, at):
    op = f"hilberta_hip::{name.split()[0]} has no derivative for torch.func"
    with pytest.raises(RuntimeError, match=op):
        torch.func.grad(lambda t: call(t).float().sum())(at)
    with pytest.raises(RuntimeError, match=op):
        torch.func.vjp(call, at)
    with pytest.raises(NotImplementedError, match="does not support it"):
        torch.func.jvp(call, (at,), (at,))


@pytest.mark.parametrize("name", NAMES)
def test_derivatives_by_transforms_are_refused(name):
    call, at = _calls("cpu")[name]
    with pytest.raises(ValueError, match="device tensors"):  # (the call itself passes every check but the last)
        call(at)
    _refused(name, call, at)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_derivatives_by_transforms_are_refused_on_the_device(name, hip_device):
    call, at = _calls(hip_device)[name]
    assert not call(at).any()
    _refused(name, call, at)
