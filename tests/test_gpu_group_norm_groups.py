"""flux_norm.group_norm of more groups than a workgroup has threads, up to one a channel of 8192 (76 KB of LDS in the second
launch), against the definition in 64 bits."""

import pytest
import torch

from hilberta_amd.flux_norm import group_norm
from oracle import layer_ops as L

pytestmark = pytest.mark.gpu
FLOAT = torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


def _normal(*shape, dtype=torch.bfloat16, std=1.0, mean=0.0):
    gen = torch.Generator("cuda").manual_seed(sum(shape))
    return (mean + std * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


# One thread joins all of a group's chunks here, up to 256 of them, after at most 20 pixels and 6 threads' sums.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, FLOAT])
@pytest.mark.parametrize("B, P, C, G", [(1, 3000, 300, 300), (2, 4100, 512, 512), (1, 3000, 1000, 1000), (1, 4300, 2000, 500), (1, 5000, 1018, 509),
                                        (1, 2100, 8192, 8192), (2, 2100, 8190, 8190), (1, 2300, 8192, 4096)])
def test_sizes(B, P, C, G, dtype):
    x = _normal(B, P, C, dtype=FLOAT)
    x = (x * _normal(C, dtype=FLOAT, mean=1.0, std=0.2) + 2 * _normal(1, C, dtype=FLOAT)).to(dtype)
    w, b = _normal(C, dtype=dtype, mean=1.0, std=0.1), _normal(C, dtype=dtype, std=0.1)
    for act in (None, "silu"):
        got, (exact, bound) = group_norm(x, G, w, b, act=act), L.group_norm(x, G, w, b, act, steps=280)
        ok = L.held(got, exact, bound)
        assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} values off, first at {(~ok).nonzero()[0].tolist()}"
        if dtype != FLOAT:
            assert L.relative(got, exact) <= torch.finfo(dtype).eps / 2
