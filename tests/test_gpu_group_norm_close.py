"""flux_norm.group_norm of few values close together far from zero, whose mean's rounding is a large part of their deviation."""

import pytest
import torch

from hilberta_amd.flux_norm import group_norm
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


# (pixels, channels, groups, roundings).  A value's difference, the missed part's, the variance's (halved by the root), the root's
# own two, and the product.  Two values: the squares' sum, its share and eps are 4, halved 2, so 8 in all and one to spare.
# Seven: their sums add 6 to the missed part's, as large as a deviation, and 6 halved to the variance's.
SIZES = [(1, 64, 32, 8), (1, 2, 1, 8), (2, 12, 12, 8), (7, 5, 5, 17)]


@pytest.mark.parametrize("mean", [0.0, 10.0, 1000.0, -30000.0])
@pytest.mark.parametrize("P, C, G, roundings", SIZES)
def test_close_values(P, C, G, roundings, mean):
    x = mean + torch.randn(40, P, C, generator=torch.Generator("cuda").manual_seed(P * C), device="cuda")
    got, (exact, bound) = group_norm(x, G), L.group_norm(x, G)
    assert L.held(got, exact, bound).all()
    assert L.relative(got, exact) <= roundings * L.U


@pytest.mark.parametrize("P", [50, 9000])
def test_the_smallest_eps(P):
    x, b = torch.full((1, P, 32), 3.25, device="cuda"), torch.randn(32, device="cuda")
    assert torch.equal(group_norm(x, 4, None, b, eps=2.0**-126), b.expand(1, P, 32))
