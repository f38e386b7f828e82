"""The quantized transformer's blocks on the GPU against their plain form in 64 bits (oracle/int8_blocks.py), each on
what it was given in a whole evaluation.  tests/int8_blocks.py derives how near they have to be, and
tests/test_int8_blocks.py shows that each mistake in their wiring is further off than that."""

import pytest
import torch

from hilberta_amd.flux_int8 import Int8Rows
from oracle import int8_blocks as B
from oracle import int8_ops as O
from tests.helpers import say
from tests.int8_blocks import BOUND, Attention, off, raise_parameters

pytestmark = pytest.mark.gpu


def _model(layers, dtype=torch.bfloat16, raised=True, **more):
    from hilberta_amd.flux_model import FluxShape, FluxTransformer

    shape = FluxShape(num_layers=layers[0], num_single_layers=layers[1], heads=4, **more)
    model = FluxTransformer("cuda", shape, seed=1, dtype=dtype)
    if raised:
        gen = torch.Generator(device="cuda").manual_seed(3)
        for w in (*model.double, *model.single, dict(norm_out=model.norm_out)):
            raise_parameters(w, gen)
        for w in model.double:
            w["norm_q"].mul_(-1)  # (raise_parameters gives every norm the same mean)
            w["norm_k"].mul_(-1)
    return model


def _inputs(model, grid, text, batch):
    from hilberta_amd.flux_model import synthetic_inputs

    args = synthetic_inputs("cuda", shape=model.shape, grid=grid, batch=batch, text_tokens=text, seed=2)
    args["timestep"] = torch.linspace(0.2, 0.9, batch, device="cuda")
    return args


def _value(rows):
    """What Int8Rows stand for; of a pair the joint rows."""
    if not isinstance(rows, Int8Rows):
        return torch.cat([_value(r) for r in rows], 1)
    return rows.q[..., :rows.features].double() * rows.scale.double()[..., None]


def _near(what, got, want):
    err = off(got, want)
    say(f"  {what}: {err:.2e}")
    assert got.shape == want.shape and err <= BOUND, what


def _mods(model, args):
    with torch.inference_mode():
        return model._modulations(model.temb(args["timestep"], args["guidance"], args["pooled_projections"], silu=True))


def _tables(args):
    from hilberta_amd.flux_inputs import rotary_tables

    return rotary_tables(torch.cat([args["txt_ids"], args["img_ids"]]))


def _embedded(model, args):
    return [torch.nn.functional.linear(args[k].to(model.dtype), *w)
            for k, w in (("hidden_states", model.x_embedder), ("encoder_hidden_states", model.context_embedder))]


@pytest.mark.parametrize("layers,grid,text,batch,dtype", [((2, 3), 8, 13, 2, torch.bfloat16), ((1, 1), 12, 77, 1, torch.float16),
                                                          ((3, 1), 6, 40, 3, torch.bfloat16)])
def test_every_block_of_an_evaluation(layers, grid, text, batch, dtype):
    model = _model(layers, dtype).quantize()
    args = _inputs(model, grid, text, batch)
    seen = []

    def spy(name, block):
        def call(w, mods, *rest):
            *before, cos, sin, attention, layer, following = rest if name == "single" else rest[:-1]
            before = [b.clone() if isinstance(b, torch.Tensor) else b for b in before]
            done = block(w, mods, *rest)
            residual = done[::2] if name == "double" else done[:1]
            if name == "double" and done[0] is None:
                residual = (rest[-1][:, text:], rest[-1][:, :text])
            seen.append((name, w, layer, before, [None if r is None else r.clone() for r in residual],
                         done[1::2] if name == "double" else done[1]))
            return done
        return call

    model._double_block_int8 = spy("double", model._double_block_int8)
    model._single_block_int8 = spy("single", model._single_block_int8)
    attention = Attention()
    prediction = model(**args, attention=attention)
    blocks = sum(layers)
    assert attention.layers == list(range(blocks)) == [s[2] for s in seen]
    double_mods, single_mods, out_mods = _mods(model, args)
    cos, sin = _tables(args)
    heads, eps = model.shape.heads, model.shape.eps
    first = [tuple(m[:2] for m in pair) for pair in double_mods] + [(m[:2], m[:2]) for m in single_mods]
    x, c = _embedded(model, args)
    for value, rows, m, s in ((x, seen[0][3][1], first[0][0], "image"), (c, seen[0][3][3], first[0][1], "text")):
        _near(f"first {s} rows", _value(rows), B.held8(O.adaln(value, *m, eps=eps)[0]))
    for i, (name, w, layer, before, residual, rows) in enumerate(seen):
        given = []
        attend = lambda *h: given.extend(h) or B.attend(*h)  # noqa: E731, B023
        if name == "double":
            assert w is model.double[i]
            (bx, bxn, bc, bcn) = before
            px, pxn, pc, pcn = B.double_block(w, double_mods[i], bx, _value(bxn), bc, _value(bcn), cos, sin, first[i + 1], heads, eps,
                                              attend)
            _near(f"block {i} image update", residual[0].double() - bx.double(), px.double() - bx.double())
            _near(f"block {i} text update", residual[1].double() - bc.double(), pc.double() - bc.double())
            _near(f"block {i} image rows", _value(rows[0]), pxn)
            _near(f"block {i} text rows", _value(rows[1]), pcn)
            after = (residual[0], rows[0], residual[1], rows[1])
        else:
            j = i - layers[0]
            assert w is model.single[j]
            bh, bhn, T = before
            following = first[i + 1][0] if i + 1 < blocks else out_mods
            ph, m = B.single_block(w, single_mods[j], bh, _value(bhn), T, cos, sin, following, heads, eps, attend)
            assert T == text
            if i + 1 < blocks:
                update, want = residual[0].double() - bh.double(), ph.double() - bh.double()
                _near(f"block {i} text update", update[:, :T], want[:, :T])
                _near(f"block {i} image update", update[:, T:], want[:, T:])
                _near(f"block {i} rows", _value(rows), B.held8(m))
            else:
                _near(f"block {i} image rows", rows, m[:, T:])
                out = (rows.double().flatten(0, 1) @ model.proj_out[0].double().t()).unflatten(0, rows.shape[:2])
                assert off(prediction, out + model.proj_out[1].double()) <= 2.0**-8
            after = (residual[0], rows)
        for got, want, s in zip(attention.given[i], given, "QKV"):
            for part, where in ((slice(0, text), "text"), (slice(text, None), "image")):
                _near(f"block {i} {where} {s}", got[:, part], want[:, part])
        if i + 1 < blocks:  # (the next block is given what this one made)
            _same_rows(name, seen[i + 1][0], after, seen[i + 1][3])


def _same_rows(name, following, after, before):
    if name == following:
        for a, b in zip(after, before):
            assert torch.equal(_value(a), _value(b)) if isinstance(a, tuple) else torch.equal(a, b)
        return
    x, xn, c, cn = after
    assert torch.equal(before[0], torch.cat([c, x], 1)) and torch.equal(_value(before[1]), torch.cat([_value(cn), _value(xn)], 1))


@pytest.mark.parametrize("batch,text", [(1, 5), (2, 13)])
def test_blocks_without_single_ones(batch, text):
    """The output norm follows the last double block."""
    model = _model((1, 0)).quantize()
    args = _inputs(model, 8, text, batch)
    prediction = model(**args, attention=Attention())
    (mods,), _, out_mods = _mods(model, args)
    eps, (x, c) = model.shape.eps, _embedded(model, args)
    xn, cn = (B.held8(O.adaln(r, *m[:2], eps=eps)[0]) for r, m in ((x, mods[0]), (c, mods[1])))
    x, _, _, _ = B.double_block(model.double[0], mods, x, xn, c, cn, *_tables(args), (out_mods, out_mods), model.shape.heads, eps)
    m = O.adaln(x, *out_mods, eps=eps)[0]
    out = (m.flatten(0, 1) @ model.proj_out[0].double().t()).unflatten(0, m.shape[:2])
    _near("prediction", prediction.double() - model.proj_out[1].double(), out)


def test_quantized_weights_are_the_layers():
    """quantize() holds each layer's own weight and bias."""
    model, int8 = _model((2, 2)), _model((2, 2)).quantize()

    def same(got, weight, bias):
        q, scale, _ = O.quantize(weight)
        assert torch.equal(got[0].q[:, :got[0].features].long(), q) and got[0].features == weight.shape[1]
        assert ((got[0].scale.double() - scale).abs() <= O.U * scale).all() and torch.equal(got[1], bias)

    for a, b in zip(int8.double, model.double):
        for name in ("qkv_x", "qkv_c", "out_x", "out_c"):
            same(a[name], *b[name])
        for name in ("ff_x", "ff_c"):
            for i in (0, 1):
                same(a[name][i], *b[name][i])
    for a, b in zip(int8.single, model.single):
        same(a["qkv"], *b["qkv"])
        same(a["mlp"], *b["mlp"])
        same(a["out"], torch.cat([b["out_attn"][0], b["out_mlp"][0]], 1), b["out_attn"][1])


@pytest.mark.parametrize("layers", [(2, 0), (1, 1), (2, 2)])
def test_every_8_bit_row_that_is_made_is_read(layers, monkeypatch):
    from hilberta_amd import flux_model

    model, made, read = _model(layers, raised=False).quantize(), [], []

    def rows_of(value):
        if isinstance(value, Int8Rows):
            return [value.q.data_ptr()]
        if isinstance(value, dict):
            value = list(value.values())
        return [p for v in value for p in rows_of(v)] if isinstance(value, (tuple, list)) else []

    def spy(name, into, of):
        call = getattr(flux_model, name)

        def spied(*args, **kwargs):
            done = call(*args, **kwargs)
            into.extend(rows_of(done if of == "done" else args))
            kept.append((args, done))  # (so that no address comes twice)
            return done
        monkeypatch.setattr(flux_model, name, spied)

    kept = []
    for name in ("adaln_quantize", "adaln_quantize_pair"):
        spy(name, made, "done")
    for name in ("int8_linear", "int8_linear_pair", "int8_qkv"):
        spy(name, read, "args")
    model(**_inputs(model, 8, 13, 2))
    assert made and set(made) == set(read)
