"""group_norm's launches follow from one element's sizes, whatever the batch (the workspace says which, on the CPU)."""

import pytest

from hilberta_amd import _lib


# (pixels, channels, groups, dtype): a group in a workgroup, small ones and many of them; chunks, up to all that there are
@pytest.mark.parametrize("sizes", [(16, 128, 128, 0), (1024, 512, 512, 0), (961, 65, 65, 2), (2100, 1, 1, 1), (3000, 64, 64, 0),
                                   (65536, 64, 32, 0), (65, 8192, 1, 0), (1 << 20, 256, 32, 2), (1 << 22, 128, 32, 0)])
def test_an_element_has_the_same_chunks_in_every_batch(sizes):
    workspace = _lib.load().hb_group_norm_workspace_bytes
    one = workspace(1, *sizes)
    for batch in (2, 100, 8191, 8192, 16384, 20000, 32768, 65535):
        assert workspace(batch, *sizes) == batch * one
