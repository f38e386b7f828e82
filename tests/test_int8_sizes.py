"""The most rows that a launch of the 8-bit row kernels takes: a grid holds fewer than 2^32 threads, and a wave takes
a row of up to 3072 features, four of them a workgroup of 256."""

import ctypes

import pytest
import torch

from hilberta_amd import _lib

MOST = (1 << 26) - 4  # rows of 2^24 - 1 workgroups


def _refused(match, name, *args):
    assert getattr(_lib.load(), name)(*args) == 1 and match in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("rows", [MOST + 1, MOST + 2, MOST + 3])
def test_rows_past_a_grid_are_refused(rows):
    P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    _refused("too many rows", "hb_int8_rows", 16, 0, 8, 1, rows, 8, 64, 0, 256, 512, None)
    pointers = (16, None, None, None, 16, 16, 16, 16)
    _refused("too many rows", "hb_int8_adaln", 1, 1, (I32 * 1)(rows), 8, 64, 0, 1e-6, (P * 8)(*pointers), (I64 * 8)(*(8,) * 8), None)
    _refused("too many rows", "hb_int8_adaln", 2, 1, (I32 * 2)(5, rows - 5), 8, 64, 0, 1e-6, (P * 16)(*pointers * 2),
             (I64 * 16)(*(8,) * 16), None)


@pytest.mark.gpu
def test_the_most_rows():
    from hilberta_amd.flux_int8 import adaln_quantize, quantize_rows

    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GiB of GPU memory")
    x = torch.zeros(MOST, 1, dtype=torch.bfloat16, device="cuda")
    x[-7:, 0] = torch.arange(1, 8, device="cuda")
    r = quantize_rows(x)
    assert (r.q[-7:, 0] == 127).all() and not r.q[:-7].any() and not r.q[-7:, 1:].any()
    assert torch.equal(r.scale[-7:] * 127, torch.arange(1.0, 8.0, device="cuda")) and not r.scale[:-7].any()
    del r
    # one row for all: LayerNorm of it is -1, 1, .., and shift 1 makes 0, 2, ..
    row = torch.tensor([1.0, 3.0] * 4, dtype=torch.bfloat16, device="cuda")
    shift, scale = torch.ones(1, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    r = adaln_quantize(row.expand(1, MOST, 8), shift, scale, eps=1e-20)
    want = torch.tensor([0, 127] * 4 + [0] * 56, dtype=torch.int8, device="cuda")
    assert torch.equal(r.q[0, 0], want) and (r.q[0, -5:] == want).all()
    assert (r.q.view(torch.int64)[..., 0] == want.view(torch.int64)[0]).all() and (r.scale == r.scale[0, 0]).all()
