"""The FLUX-shaped transformer with its blocks' linear layers in 8 bits (FluxTransformer.quantize).

Against the same model in 16 bits.  A row rounded to whole steps of its top / 127 is off by step / sqrt(12)
at the root mean square, top / rms / 440 of itself: 1 % for rows whose top is 4.5 times their rms (normal
values of a few thousand features), 1.8 % for 8 times (GELU's outputs).  Rounding the weights' channels adds
the same 1 % to each layer.  A block rounds its rows four times (Q/K/V, output projection, MLP in and out),
so its update is off by 1 + 1 + 1 + 1.8 and 4 x 1 %, added in squares (the roundings are independent) 3.2 %;
the updates of five blocks at most, all of them in one direction, 16 % of an update.  Updates enter the residual
stream through gates of 0.2: the stream, and the prediction, are off by less than that.
"""

import pytest
import torch

from tests.helpers import say

pytestmark = pytest.mark.gpu

REL_L2 = 0.16


def _rel(a, b):
    a, b = a.float(), b.float()
    return float((a - b).norm() / b.norm())


def _models(device, **shape):
    """The same model in 16 and in 8 bits, and inputs."""
    from hilberta_amd.flux_model import FluxShape, FluxTransformer, synthetic_inputs

    shape = FluxShape(**shape)
    return (FluxTransformer(device, shape, seed=1), FluxTransformer(device, shape, seed=1).quantize(),
            lambda **kw: synthetic_inputs(device, shape=shape, seed=2, **kw))


def test_prediction_near_the_16_bit_model(hip_device):
    from hilberta_amd.bridge_k import paired_plan_device
    from hilberta_amd.flux_model import NativeAttention, PersistentAttention

    model, int8, inputs = _models(hip_device, num_layers=2, num_single_layers=3, heads=4)
    assert int8.quantize() is int8  # (again: nothing)
    args = inputs(grid=64)
    paired = PersistentAttention(paired_plan_device(4, 1, grid_size=64, device=hip_device), hip_device)
    for name, attention in (("paired", paired), ("native", NativeAttention())):
        want, got = model(**args, attention=attention), int8(**args, attention=attention)
        torch.cuda.synchronize()
        err = _rel(got, want)
        say(f"  {name}: relative L2 {err:.3e}")
        assert got.shape == want.shape and got.dtype == want.dtype and err <= REL_L2
        assert err > 1e-4  # (the 8-bit layers ran)
        assert torch.equal(got, int8(**args, attention=attention))
    assert paired.calls == 15


@pytest.mark.parametrize("layers", [(1, 0), (1, 1), (2, 1)])
def test_other_depths(hip_device, layers):
    model, int8, inputs = _models(hip_device, num_layers=layers[0], num_single_layers=layers[1], heads=4)
    args = inputs(grid=16, text_tokens=77)
    assert _rel(int8(**args), model(**args)) <= REL_L2


def test_batch_equals_its_elements(hip_device):
    """Sums are whole numbers, so only the 16-bit layers around the blocks (embedders, modulations, output)
    may round differently with the batch."""
    _, int8, inputs = _models(hip_device, num_layers=1, num_single_layers=1, heads=4)
    args = inputs(grid=16, batch=3, text_tokens=40)
    together = int8(**args)
    for b in range(3):
        one = {k: v if k.endswith("_ids") else v[b:b + 1] for k, v in args.items()}
        assert _rel(together[b:b + 1], int8(**one)) <= 2e-2


def test_half_the_weights(hip_device):
    model, int8, _ = _models(hip_device, num_layers=1, num_single_layers=1, heads=4)
    size = lambda m: sum(p.numel() * p.element_size() for p in m.parameters() if p is not None)  # noqa: E731
    assert size(int8) < 0.8 * size(model)  # (embedders and modulations stay)


def test_no_double_blocks_is_refused(hip_device):
    from hilberta_amd.flux_model import FluxShape, FluxTransformer

    with pytest.raises(ValueError, match="without double blocks"):
        FluxTransformer(hip_device, FluxShape(num_layers=0, num_single_layers=1, heads=4)).quantize()
