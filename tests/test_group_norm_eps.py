"""group_norm's eps: what the kernels' root would take for zero is refused (CPU)."""

import pytest
import torch

from hilberta_amd import _lib
from hilberta_amd.flux_norm import group_norm


@pytest.mark.parametrize("eps", [0.0, -1e-6, 1.1e-38, 1e-40, 1e-50, float("nan")])
def test_refused(eps):
    with pytest.raises(ValueError, match="eps must be at least"):
        group_norm(torch.zeros(2, 6, 8), 4, eps=eps)
    held = 1 << 40  # (an address that nothing reads)
    assert _lib.load().hb_group_norm(1, 6, 8, 4, 2, 0, eps, held, 48, 8, None, None, held, 48, 8, None, 0, None) == 1
    assert b"eps must be at least" in _lib.load().hb_last_error()


@pytest.mark.parametrize("eps", [2.0**-126, 1e-6, 1.0])
def test_taken(eps):
    with pytest.raises(ValueError, match="device tensors"):
        group_norm(torch.zeros(2, 6, 8), 4, eps=eps)
