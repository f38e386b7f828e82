"""flux_norm.group_norm on the CPU: what it refuses, and that it runs nowhere but on the GPU."""

import pytest
import torch

from hilberta_amd.flux_norm import group_norm

ON_DEVICE = "device tensors"


def _refused(match, x, groups=4, *args, **kwargs):
    with pytest.raises(ValueError, match=match):
        group_norm(x, groups, *args, **kwargs)


def _image(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).contiguous(memory_format=torch.channels_last if len(shape) == 4 else torch.channels_last_3d)


def test_a_call_that_passes_every_check_needs_the_gpu():
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _refused(ON_DEVICE, torch.zeros(2, 6, 8, dtype=dtype))
        _refused(ON_DEVICE, _image(2, 8, 3, 5, dtype=dtype), act="silu")
        _refused(ON_DEVICE, _image(2, 8, 2, 3, 5, dtype=dtype), 8, torch.zeros(8, dtype=dtype), torch.zeros(8, dtype=dtype))
    x = torch.zeros(2, 6, 8)
    _refused(ON_DEVICE, x, out=x)
    _refused(ON_DEVICE, x, out=torch.empty_like(x))
    _refused(ON_DEVICE, torch.zeros(2, 0, 8))
    _refused(ON_DEVICE, torch.zeros(2, 8, 1, 1))
    _refused(ON_DEVICE, torch.zeros(2, 9, 12)[:, 2:5, 1:9])
    _refused(ON_DEVICE, _image(2, 12, 4, 6)[:, 2:10])
    _refused(ON_DEVICE, _image(2, 8, 4, 6)[:, :, 1:3])


def test_shapes_and_types():
    x = torch.zeros(2, 6, 8)
    _refused("act must be", x, act="gelu")
    _refused("x must be bf16", x.double())
    _refused("x must be", x[0])
    _refused("x must be", x[None, None, None])
    _refused("groups must divide", x, 3)
    _refused("groups must divide", x, 0)
    _refused("1 to 8192", torch.zeros(1, 1, 8196))
    _refused("1 to 8192", torch.zeros(1, 1, 0))
    _refused("eps must be", x, eps=0.0)
    _refused("channels last", torch.zeros(2, 8, 3, 5))
    _refused("channels last", x.transpose(1, 2).contiguous().transpose(1, 2))
    _refused("evenly apart", _image(2, 8, 4, 6)[..., :5])
    for w in (torch.zeros(7), torch.zeros(8, dtype=torch.bfloat16), torch.zeros(16)[::2], torch.zeros(1, 8)):
        _refused("weight and bias", x, 4, w)
        _refused("weight and bias", x, 4, None, w)
    _refused("out must be like x", x, out=torch.zeros(2, 6, 9))
    _refused("out must be like x", x, out=torch.zeros(2, 6, 8, dtype=torch.bfloat16))


def test_what_is_written_lies_apart():
    x = torch.zeros(3, 6, 8)
    _refused("cannot alias", x[:2], out=x[1:])
    _refused("cannot alias", x, 4, x[0, 0], out=x)
    _refused("non-overlapping", x, out=torch.zeros(1, 6, 8).expand(3, 6, 8))


def test_gradients_are_refused():
    w = torch.zeros(8, requires_grad=True)
    _refused("Inference only", torch.zeros(2, 6, 8), 4, w)
    with torch.no_grad():
        _refused(ON_DEVICE, torch.zeros(2, 6, 8), 4, w)
    with pytest.raises(RuntimeError, match="group_norm has no derivative for torch.func"):
        torch.func.grad(lambda x: group_norm(x, 4).sum())(torch.zeros(2, 6, 8))


def test_shapes_of_traced_calls():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        y = group_norm(torch.empty(2, 8, 4, 6, device="cuda", memory_format=torch.channels_last), 4, act="silu")
        assert y.shape == (2, 8, 4, 6) and y.is_contiguous(memory_format=torch.channels_last)
        assert group_norm(torch.empty(2, 24, 8, device="cuda"), 4).shape == (2, 24, 8)


# ------------------------------------------------------------------ the C entry (addresses that nothing reads)
def test_workspaces():
    import ctypes

    from hilberta_amd import _lib

    lib, held = _lib.load(), ctypes.c_void_p(1 << 40)

    def call(sizes, workspace, bytes):
        batch, pixels, channels, *_ = sizes
        return lib.hb_group_norm(*sizes, 0, 1e-6, held, pixels * channels, channels, None, None, held, pixels * channels, channels,
                                 workspace, bytes, None)

    assert lib.hb_group_norm_workspace_bytes(1, 256, 512, 32, 0) == 0  # (a workgroup holds a group)
    sizes = (2, 16384, 512, 32, 0)
    need = lib.hb_group_norm_workspace_bytes(*sizes)
    assert need > 0 and need == 2 * lib.hb_group_norm_workspace_bytes(1, *sizes[1:])
    for workspace, bytes in ((None, need), (held, need - 1), (ctypes.c_void_p((1 << 40) + 4), need)):
        assert call(sizes, workspace, bytes) == 1 and b"the workspace must hold" in lib.hb_last_error()
    for sizes in ((0, 9, 8, 4, 0), (65536, 9, 8, 4, 0), (1, 0, 8, 4, 0), (1, 1 << 31, 8, 4, 0), (1, 9, 8193, 1, 0), (1, 9, 0, 1, 0),
                  (1, 9, 8, 3, 0), (1, 9, 8, 0, 0), (1, 9, 8, 4, 3), (1, 9, 8, 4, -1)):
        assert lib.hb_group_norm_workspace_bytes(*sizes) == -1
        assert call(sizes, held, 1 << 20) == 1
