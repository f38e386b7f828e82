"""flux_linear on the CPU: what its operators refuse, and that they run nowhere but on the GPU.

The operators make their checks on any device and refuse CPU tensors last: a call that passes every check ends with
that refusal.
"""

import ctypes

import pytest
import torch

from hilberta_amd import _lib, ops
from hilberta_amd import flux_linear as f

BF16, HALF = torch.bfloat16, torch.float16
ON_DEVICE = "device tensors"
B, M, K, N = 2, 3, 24, 40


def _args(**changes):
    a = dict(x=torch.zeros(B, M, K, dtype=BF16), weight=torch.zeros(N, K, dtype=BF16), bias=torch.zeros(N, dtype=BF16),
             residual=torch.zeros(B, M, N, dtype=BF16), gate=torch.zeros(B, N, dtype=BF16))
    return {k: v for k, v in (a | changes).items() if v is not None or k in ("bias", "residual", "gate")}


def _refused(match, **changes):
    with pytest.raises(ValueError, match=match):
        f.linear(**_args(**changes))


def test_a_call_that_passes_every_check_needs_the_gpu():
    for changes in ({}, dict(bias=None), dict(gate=None), dict(gate=None, residual=None), dict(act="gelu"), dict(act="silu"),
                    dict(out=torch.zeros(B, M, N, dtype=BF16)),
                    dict(x=torch.zeros(M, K, dtype=BF16), residual=torch.zeros(M, N, dtype=BF16), gate=torch.zeros(1, N, dtype=BF16)),
                    dict(x=torch.zeros(B, 0, K, dtype=BF16), residual=torch.zeros(B, 0, N, dtype=BF16)),
                    dict(x=torch.zeros(B, M, K + 8, dtype=BF16)[..., 3:3 + K], weight=torch.zeros(N, K + 5, dtype=BF16)[:, 1:1 + K])):
        _refused(ON_DEVICE, **changes)


def test_shapes_and_types():
    zeros = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    _refused("act must be", act="relu")
    _refused("act must be", act=True)
    _refused("x must be", x=zeros(K))
    _refused("x must be", weight=zeros(N))
    _refused("x must be", x=zeros(B, 1, M, K))
    _refused("weight must be", weight=zeros(N, K + 1))
    _refused("weight must be", weight=zeros(K, N).T)
    _refused("weight must be", x=zeros(B, M, 0), weight=zeros(N, 0))
    _refused("contiguous last dimension", x=zeros(B, K, M).transpose(1, 2))
    _refused("bias must be", bias=zeros(N + 1))
    _refused("bias must be", bias=zeros(2 * N)[::2])
    _refused("residual must be like out", residual=zeros(B, M, N + 1))
    _refused("residual must have a contiguous", residual=zeros(B, N, M).transpose(1, 2))
    _refused("needs its residual", residual=None)
    _refused("gate must be", gate=zeros(B + 1, N))
    _refused("gate must be", gate=zeros(N))
    _refused("gate must be", gate=zeros(N, B).T)
    _refused("out must be", out=zeros(B, M, N + 1))
    for name, shape in (("weight", (N, K)), ("bias", (N,)), ("residual", (B, M, N)), ("gate", (B, N)), ("out", (B, M, N))):
        _refused("rows' dtype", **{name: zeros(*shape, dtype=HALF)})
    _refused("bf16 or fp16", x=zeros(B, M, K, dtype=torch.float32))
    with pytest.raises(ValueError, match="act must be 0"):
        ops.linear(zeros(B, M, K), zeros(N, K), None, None, None, 3)


def test_what_is_written_lies_apart():
    buffer = torch.zeros(B, M, K + N, dtype=BF16)
    _refused(ON_DEVICE, out=buffer[..., K:])
    _refused(ON_DEVICE, x=buffer[..., :K], out=buffer[..., K:])
    _refused("apart from the rows", x=buffer[..., 1:K + 1], out=buffer[..., K:])
    _refused("non-overlapping", out=torch.zeros(1, M, N, dtype=BF16).expand(B, M, N))
    res = torch.zeros(B, M, N, dtype=BF16)
    _refused(ON_DEVICE, residual=res, out=res)
    wide = torch.zeros(B, M, N + 1, dtype=BF16)
    _refused("residual itself", residual=wide[..., 1:], out=wide[..., :N])
    _refused(ON_DEVICE, residual=torch.zeros(B, M, 2 * N, dtype=BF16)[..., :N], out=res)
    both = torch.zeros(B, M, 2 * N, dtype=BF16)
    _refused(ON_DEVICE, residual=both[..., :N], out=both[..., N:])
    flat = torch.zeros(B * N, dtype=BF16)
    _refused("cannot alias", gate=flat.view(B, N), residual=torch.zeros(B, 1, N, dtype=BF16),
             x=torch.zeros(B, 1, K, dtype=BF16), out=flat.view(B, 1, N))


def test_pairs():
    a, b = _args(), _args(x=torch.zeros(B, 5, K, dtype=BF16), residual=torch.zeros(B, 5, N, dtype=BF16))

    def pair(match, **changes):
        with pytest.raises(ValueError, match=match):
            f.linear_pair(a, b | changes)

    pair(ON_DEVICE)
    pair(ON_DEVICE, x=torch.zeros(B, 0, K, dtype=BF16), residual=None, gate=None)
    pair("share batch", x=torch.zeros(B + 1, 5, K, dtype=BF16), residual=None, gate=None)
    pair("share batch", weight=torch.zeros(N + 8, K, dtype=BF16), bias=None, residual=None, gate=None)
    pair("share batch", x=torch.zeros(B, 5, K + 8, dtype=BF16), weight=torch.zeros(N, K + 8, dtype=BF16))
    out = torch.zeros(B, 8, N, dtype=BF16)
    with pytest.raises(ValueError, match=ON_DEVICE):
        f.linear_pair(a | dict(out=out[:, :3]), b | dict(out=out[:, 3:]))
    with pytest.raises(ValueError, match="lie apart"):
        f.linear_pair(a | dict(out=out[:, :3]), b | dict(out=out[:, 2:7]))
    with pytest.raises(ValueError, match="residual itself"):  # (one set's output over the other's residual)
        f.linear_pair(a | dict(out=b["residual"][:, :3]), b)


def test_gradients_are_refused():
    a = _args(weight=torch.zeros(N, K, dtype=BF16, requires_grad=True))
    with pytest.raises(ValueError, match="Inference only"):
        f.linear(**a)
    with torch.no_grad(), pytest.raises(ValueError, match=ON_DEVICE):
        f.linear(**a)
    with pytest.raises(RuntimeError, match="linear has no derivative for torch.func"):
        torch.func.grad(lambda w: f.linear(_args()["x"], w).float().sum())(_args()["weight"])
    with pytest.raises(NotImplementedError, match="does not support it"):
        torch.func.jvp(lambda w: f.linear(_args()["x"], w), (_args()["weight"],), (_args()["weight"],))


def test_shapes_of_traced_calls():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(2, 5, 24, dtype=HALF, device="cuda"), torch.empty(40, 24, dtype=HALF, device="cuda")
        y = f.linear(x, w, act="silu")
        assert y.shape == (2, 5, 40) and y.dtype == HALF and y.device.type == "cuda"
        assert [t.shape[1] for t in f.linear_pair(dict(x=x, weight=w), dict(x=x[:, :3], weight=w))] == [5, 3]


# ------------------------------------------------------------------ the C entry (addresses that nothing reads)
HELD = 1 << 40


def _workspace(rows, columns, features, *, x=HELD, row=None, count=1, batch=1):
    pointers = (ctypes.c_void_p * 12)(*([x, HELD, None, None, None, HELD] * 2))
    row = features if row is None else row
    strides = (ctypes.c_int64 * 16)(*([rows * row, row, features, 0, 0, 0, rows * columns, columns] * 2))
    call = (count, batch, (ctypes.c_int32 * 2)(rows, rows), columns, features)
    return _lib.load().hb_linear_workspace_bytes(*call, pointers, strides), call, pointers, strides


def test_workspaces():
    # whole tiles, or enough of them: nothing
    for rows, columns, features in ((4096, 9216, 3072), (1, 18432, 3072), (16, 5, 1001), (77, 64, 64)):
        assert _workspace(rows, columns, features)[0] == 0
    # few tiles over many features: the sums of parts of them
    for rows, columns, features in ((126, 32, 13952), (100, 304, 12288), (512, 3072, 12288), (8, 512, 12288)):
        parts = _workspace(rows, columns, features)[0] / (rows * columns * 4)
        assert parts in (2, 3, 4, 6, 8, 12, 16)
    assert _workspace(126, 27, 13952)[0] % (126 * 32 * 4) == 0
    # rows and weights that direct loads cannot take (their strides, their address, too far apart), where copies pay
    both, rows = 7000 * 5056 * 2, 2000 * 5056 * 2
    assert _workspace(2000, 5000, 5001)[0] == both and _workspace(2000, 5000, 5001, count=2)[0] == 2 * both
    assert _workspace(2000, 5000, 5056, x=HELD + 2)[0] == rows
    assert _workspace(2000, 5000, 5056, row=5057)[0] == rows
    assert _workspace(2000, 5000, 5056, row=1 << 23)[0] == rows
    assert _workspace(2000, 5000, 3)[0] == 7000 * 64 * 2  # (rows of fewer than eight)
    # and where they do not
    for size in ((300, 1000, 60), (999, 777, 1001), (2405, 20, 13)):
        assert _workspace(*size)[0] == 0
    for bad in (dict(rows=0), dict(columns=0), dict(features=0), dict(features=(1 << 20) + 1), dict(columns=(1 << 25) + 1), dict(count=0), dict(count=3), dict(batch=0),
                dict(x=None), dict(x=HELD + 1), dict(row=-8)):
        assert _workspace(**(dict(rows=300, columns=1000, features=64) | bad))[0] == -1


def test_a_workspace_too_small_is_refused():
    for sizes in ((126, 32, 13952), (2000, 5000, 5001)):
        bytes, call, pointers, strides = _workspace(*sizes)
        assert bytes > 0
        for workspace, held in ((None, bytes), (HELD, bytes - 1), (HELD + 8, bytes)):
            assert _lib.load().hb_linear(*call, 0, 0, pointers, strides, workspace, held, None) == 1
            assert b"the workspace must hold" in _lib.load().hb_last_error()
    for dtype, act, match in ((2, 0, b"dtype must be"), (0, 3, b"act must be")):
        bytes, call, pointers, strides = _workspace(1, 8, 8)
        assert _lib.load().hb_linear(*call, dtype, act, pointers, strides, None, 0, None) == 1
        assert match in _lib.load().hb_last_error()
