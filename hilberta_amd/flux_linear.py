"""Linear layers in 16 bits with what follows them in the same pass (csrc/linear.hip).

``linear(x, weight, bias, act=act, residual=residual, gate=gate)`` computes, per row,

    out = residual + gate * act(x @ weight^T + bias)

for a caller's own layers (FluxTransformer has library products or 8-bit ones), which a transformer block runs as a library product and one to three passes over its output
(``F.linear``, an activation, ``torch.addcmul``), and an image decoder as a convolution of one pixel and an
addition.  Sums and epilogue are fp32, rounded once to the 16-bit output.  ``linear_pair`` does so for two row
sets with weights of their own (a block's text and image rows) in one launch.

Inference only: inputs that need a gradient are refused.  Launches are asynchronous on the current stream and can
be captured into a graph.  Rows, weights and outputs may be row ranges or column blocks of larger buffers; rows
that are no multiple of 16 bytes may be copied into aligned ones first, weights in every call (a caller that keeps one
pads its features and the rows' to a multiple of eight, with zeros), and a long sum for few outputs is made in
parts, joined in their order; both take a workspace for the call.  A layer of one or two rows is read faster by
flux_cond.linear_layers, which takes many layers at once.  The reference has library calls here (in the
transformer that hilberta/flux_adapter.py wraps).
"""

from __future__ import annotations

import torch

from . import ops

_ACTS = {None: 0, "gelu": 1, "silu": 2}


def _act(act):
    if act not in _ACTS:
        raise ValueError('act must be None, "gelu" (tanh) or "silu"')
    return _ACTS[act]


def linear(x, weight, bias=None, *, act=None, residual=None, gate=None, out=None):
    """residual + gate * act(x @ weight^T + bias) for x [rows, features] or [B, rows, features].

    weight [out_features, features] and bias [out_features]; act None, "gelu" (tanh) or "silu"; residual like
    the output, gate [B, out_features] (only with a residual; B is 1 for two-dimensional x).  All in one 16-bit
    dtype, with contiguous last dimensions.  ``out`` may be the residual itself, for an update in place."""
    if out is None:
        return ops.linear(x, weight, bias, residual, gate, _act(act))
    ops.linear_out(x, weight, bias, residual, gate, out, _act(act))
    return out


def _set(x, weight, bias=None, residual=None, gate=None, out=None):
    return (x, weight, bias, residual, gate), out


def linear_pair(first, second, *, act=None):
    """linear of two row sets in one launch: ``first`` and ``second`` are dicts of x, weight, bias, residual,
    gate and out, of one batch, layer shape, dtype and device; either may have no rows.  Returns both outputs."""
    (a, out_a), (b, out_b) = _set(**first), _set(**second)
    if out_a is None and out_b is None:
        return ops.linear_pair(*a, *b, _act(act))
    if out_a is None or out_b is None:
        x, weight = (a if out_a is None else b)[:2]
        made = torch.empty(*x.shape[:-1], weight.shape[0], dtype=x.dtype, device=x.device)
        out_a, out_b = (made, out_b) if out_a is None else (out_a, made)
    ops.linear_pair_out(*a, out_a, *b, out_b, _act(act))
    return out_a, out_b
