"""flux_norm.group_norm of batches that take several launches: an image's result is the same as alone, bit for bit."""

import pytest
import torch

from hilberta_amd.flux_norm import group_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu(hip_device):
    return hip_device


def _normal(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(sum(shape)), device="cuda").to(dtype)


def test_many_small_groups():
    """More groups in all than one launch of full workgroups would take; these are small."""
    x = _normal(32768, 16, 128)
    got = group_norm(x, 128, act="silu")
    for i in (0, 1, 4095, 20000, 32767):
        assert torch.equal(got[i:i + 1], group_norm(x[i:i + 1], 128, act="silu"))
    assert torch.equal(got[-300:], group_norm(x[-300:], 128, act="silu"))


def test_groups_of_a_workgroup_in_two_launches():
    """65 groups of 1024 threads by 65535 elements: 2^32 threads and more."""
    x = _normal(1, 961, 65)
    want = group_norm(x, 65, act="silu")
    got = group_norm(x.expand(65535, -1, -1), 65, act="silu")
    assert all((part == want).all() for part in got.split(8192))


def test_chunks_in_two_launches():
    """65 chunks of 1024 threads by 65535 elements; 70 GB of outputs, past 2^35 of them."""
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of free memory")
    x = _normal(1, 65, 8192)
    want = group_norm(x, 2, act="silu")
    got = group_norm(x.expand(65535, -1, -1), 2, act="silu")
    assert all((part == want).all() for part in got.split(2048))
    del got
    torch.cuda.empty_cache()
