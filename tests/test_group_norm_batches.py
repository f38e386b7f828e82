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


# (pixels, channels, dtype, chunks, or one fewer where the last would be empty): twice the chunks only where they are faster
@pytest.mark.parametrize("pixels, channels, dtype, chunks", [
    (1 << 21, 128, 0, 256), (5 << 19, 128, 0, 512), (1 << 22, 128, 1, 512), (9 << 17, 128, 2, 256), (1 << 21, 128, 2, 512),
    (1 << 26, 8, 0, 512), (8947848, 60, 0, 256), (5592405, 96, 1, 256), (4473924, 60, 2, 256), (1677721, 320, 0, 512),
    (535799, 1002, 0, 512), (89478485, 6, 0, 512)])
def test_chunks_of_large_elements(pixels, channels, dtype, chunks):
    bytes = _lib.load().hb_group_norm_workspace_bytes(1, pixels, channels, 1, dtype)
    assert bytes // 8 in (chunks, chunks - 1)
