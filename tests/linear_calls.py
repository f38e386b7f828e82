"""What hb_linear would run for a call, asked of the host alone (addresses that nothing reads)."""

import ctypes

from hilberta_amd import _lib

HELD = 1 << 40
ACTS = {None: 0, "gelu": 1, "silu": 2}


def call(batch, rows, K, N, *, act=None, more="", out_row=None, shift=0, sets=None):
    """(hb_linear_choice's four numbers, hb_linear_workspace_bytes) of contiguous operands; `rows` of one set or two, `more`
    "", "residual", "gate" or one of them a set; outputs `out_row` apart that begin `shift` elements past 16 bytes."""
    rows = (rows,) if isinstance(rows, int) else rows
    more = (more,) * len(rows) if isinstance(more, str) else more
    out_row = N if out_row is None else out_row
    pointers, strides = [], []
    for m, kind in zip(rows, more):
        pointers += [HELD, HELD, HELD, HELD if kind else None, HELD if kind == "gate" else None, HELD + 2 * shift]
        strides += [m * K, K, K, m * N, N, N, m * out_row, out_row]
    args = (len(rows), batch, (ctypes.c_int32 * 2)(*rows), N, K)
    p, s = (ctypes.c_void_p * 12)(*pointers), (ctypes.c_int64 * 16)(*strides)
    choice, lib = (ctypes.c_int32 * 4)(), _lib.load()
    assert lib.hb_linear_choice(*args, ACTS[act], p, s, choice) == 0, _lib.last_error()
    return tuple(choice), lib.hb_linear_workspace_bytes(*args, p, s)


# (batch, rows of one set or two, features, columns) that the wide kernel takes in one part and finishes through LDS: tiles
# of several batch elements, columns that are no multiple of eight
GENERAL = [(3, 1365, 512, 4096), (3, 1365, 776, 4089), (32, 128, 776, 4096), (315, 13, 776, 4089), (1, 4096, 1032, 4094)]
GENERAL_PAIRS = [(3, (700, 1365), 520, 4096), (3, (700, 1365), 520, 4091), (16, (112, 144), 520, 4092)]
SHIFTS = [(0, 0), (1, 13), (2, 12)]  # outputs that many elements past 16 bytes, with rows so much longer
