"""Row sets without rows: the forms of two sets take them as those of one set do, with the same checks."""

import pytest
import torch

from hilberta_amd import flux_int8 as f

BF16 = torch.bfloat16
ON_DEVICE = "device tensors"


def _refused(match, call, *args, **kwargs):
    with pytest.raises(ValueError, match=match):
        call(*args, **kwargs)


def _rows(*lead, features=70, device="cpu"):
    q = torch.zeros(*lead, f.padded_features(features), dtype=torch.int8, device=device)
    return f.Int8Rows(q, torch.zeros(lead, device=device), features, BF16)


def _weight(columns, features=70, device="cpu"):
    q = torch.zeros(columns, f.padded_features(features), dtype=torch.int8, device=device)
    return f.Int8Weight(q, torch.zeros(columns, device=device), features)


def test_checks_come_before_an_empty_result():
    """(The refusal of CPU tensors is the last check.)"""
    w, b = _weight(5), torch.zeros(5, dtype=BF16)
    _refused(ON_DEVICE, f.int8_linear, _rows(0), w, b)
    _refused("bias", f.int8_linear, _rows(0), w, b[:4])
    _refused("as the rows are padded", f.int8_linear, _rows(0), f.Int8Weight(torch.zeros(5, 192, dtype=torch.int8), torch.zeros(5), 70))
    for n, m in ((0, 3), (3, 0), (0, 0)):
        _refused(ON_DEVICE, f.int8_linear_pair, dict(x=_rows(2, n), weight=w), dict(x=_rows(2, m), weight=w, bias=b))
        _refused("bias", f.int8_linear_pair, dict(x=_rows(2, n), weight=w), dict(x=_rows(2, m), weight=w, bias=b[:4]))
        x, v = torch.zeros(2, 9, 64, dtype=BF16), torch.zeros(2, 64, dtype=BF16)
        _refused(ON_DEVICE, f.adaln_quantize_pair, dict(x=x[:, :n], shift=v, scale=v), dict(x=x[:, :m], shift=v, scale=v))
        _refused("shift/scale", f.adaln_quantize_pair, dict(x=x[:, :n], shift=v, scale=v), dict(x=x[:, :m], shift=v, scale=v[:1]))


@pytest.mark.gpu
def test_checks_come_before_an_empty_result_on_the_device():
    w, b = _weight(5, device="cuda"), torch.zeros(5, dtype=BF16, device="cuda")
    assert f.int8_linear(_rows(0, device="cuda"), w, b).shape == (0, 5)
    _refused("bias", f.int8_linear, _rows(0, device="cuda"), w, b[:4])
    _refused("bias", f.int8_linear, _rows(2, 0, device="cuda"), w, b[:4], out=torch.empty(2, 0, 5, dtype=BF16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("first,second", [(0, 40), (40, 0), (0, 0)])
def test_one_of_two_sets_is_empty(first, second):
    gen = torch.Generator(device="cuda").manual_seed(first)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").to(BF16)  # noqa: E731
    B, C, N = 2, 72, 33
    w, b = f.quantize_weight(randn(N, C)), randn(N)
    xs, ys, mods = [randn(B, n, C) for n in (first, second)], [randn(B, n, C) for n in (first, second)], randn(B, 3 * C).chunk(3, 1)
    outs = [torch.full_like(x, 7.0) for x in xs]
    sets = [dict(x=x, shift=mods[0], scale=mods[1], y=y, gate=mods[2], x_out=o) for x, y, o in zip(xs, ys, outs)]
    pair = f.adaln_quantize_pair(*sets)
    for s, got, out in zip(sets, pair, outs):
        alone = torch.full_like(out, 7.0)
        want = f.adaln_quantize(**{**s, "x_out": alone})
        assert got.q.shape == (B, s["x"].shape[1], 128) and got.scale.shape == (B, s["x"].shape[1])
        assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale) and torch.equal(out, alone)
    buf = torch.full((B, 50, N), 7.0, dtype=BF16, device="cuda")
    into = dict(x=pair[1], weight=w, out=buf[:, 3:3 + second])
    one, two = f.int8_linear_pair(dict(x=pair[0], weight=w, bias=b), into, gelu=True)
    assert torch.equal(one, f.int8_linear(pair[0], w, b, gelu=True)) and two is into["out"]
    assert torch.equal(two, f.int8_linear(pair[1], w, gelu=True))
    assert (buf[:, :3] == 7).all() and (buf[:, 3 + second:] == 7).all()


@pytest.mark.gpu
def test_transformer_without_text_rows():
    """FluxTransformer.quantize's blocks on image rows alone."""
    from hilberta_amd.flux_model import FluxShape, FluxTransformer, synthetic_inputs

    shape = FluxShape(num_layers=2, num_single_layers=1, heads=4)
    model = FluxTransformer("cuda", shape, seed=1).quantize()
    args = synthetic_inputs("cuda", shape=shape, grid=8, batch=2, text_tokens=0, seed=2)
    got = model(**args)
    assert got.shape == (2, 64, 64) and torch.isfinite(got).all()
    # text rows that attention does not look at change nothing
    more = synthetic_inputs("cuda", shape=shape, grid=8, batch=2, text_tokens=3, seed=2)
    more = {**args, **{k: more[k] for k in ("encoder_hidden_states", "txt_ids")}}

    class ImageOnly:
        layout = None

        def __call__(self, layer, q, k, v, out):
            from hilberta_amd.flux_model import NativeAttention

            out.zero_()
            part = torch.empty_like(q[:, :, 3:])
            NativeAttention()(layer, q[:, :, 3:].contiguous(), k[:, :, 3:].contiguous(), v[:, :, 3:].contiguous(), part)
            out[:, :, 3:] = part

    want = model(**more, attention=ImageOnly())
    off = (got.float() - want.float()).norm() / want.float().norm()
    assert off <= 2e-2  # (16-bit layers around the blocks may round differently: as for the elements of a batch)
