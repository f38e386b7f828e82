"""Which kernel hb_linear takes (hb_linear_choice, on the CPU): the epilogue that the wide kernel would run is part of its
estimate, and the workspace holds what every activation takes."""

import random

import pytest

from tests.linear_calls import GENERAL, GENERAL_PAIRS, SHIFTS, call


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("more", ["residual", "gate"])
def test_shallow_layers_with_activation_and_residual_leave_the_wide_kernel(act, more):
    """Its tiles would go through LDS there: 32 to 36 us, where smaller ones take 9 to 10."""
    for size in ((1, 80, 64, 18048), (1, 1330, 64, 1664), (1, 10240, 128, 256)):
        assert call(*size)[0][:2] == (256, 256)
        assert call(*size, act=act, more=more)[0][:2] != (256, 256)
    # and deep ones stay on it
    assert call(1, 4096, 3072, 9216, act=act, more=more)[0] == (256, 256, 1, 1)
    assert call(1, 4096, 3072, 9216, more=more)[0] == (256, 256, 1, 0)


def test_pairs_whose_sets_differ_leave_the_wide_kernel():
    size = (2, (512, 2048), 512, 4000)
    assert call(*size)[0] == call(*size, more="gate")[0] == (256, 256, 1, 0)
    for mixed in (("", "gate"), ("gate", ""), ("residual", "gate")):
        assert call(*size, more=mixed)[0][:2] != (256, 256)


def test_the_workspace_holds_the_parts_of_every_activation():
    def check(batch, rows, K, N, more):
        for act in (None, "gelu", "silu"):
            (_, _, parts, _), bytes = call(batch, rows, K, N, act=act, more=more)
            assert parts == 1 or bytes >= parts * batch * rows * ((N + 7) // 8 * 8) * 4

    check(1, 13632, 2176, 384, "residual")  # (one part without an activation, two with one)
    rng = random.Random(3)
    for _ in range(400):
        check(rng.choice((1, 1, 3)), round(10 ** rng.uniform(0, 4)), 8 * round(10 ** rng.uniform(0, 3.2)),
              round(10 ** rng.uniform(0.5, 4)), rng.choice(("", "residual", "gate")))


def test_refusals():
    with pytest.raises(AssertionError, match="batch and rows must be positive"):
        call(1, 0, 64, 64)
    with pytest.raises(AssertionError, match="features must be"):
        call(1, 9, 0, 64)


@pytest.mark.parametrize("size", GENERAL + GENERAL_PAIRS)
def test_sizes_of_the_general_epilogue(size):
    """What tests/test_gpu_linear_general.py runs takes the route that it is about."""
    for act in (None, "gelu", "silu"):
        for more in ("", "residual", "gate"):
            for shift, longer in SHIFTS:
                assert call(*size, act=act, more=more, out_row=size[3] + longer, shift=shift)[0] == (256, 256, 1, 1)
