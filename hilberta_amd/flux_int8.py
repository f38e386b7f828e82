"""The denoiser's linear layers in 8-bit integers (csrc/int8_rows.hip, csrc/int8_gemm.hip).

Activations hold one scale a row (token), weights one a row (output channel): value = q * scale.

  quantize_rows     16-bit rows to 8-bit rows:  scale = max|x| / 127,  q = rint(127 x / max|x|)
  quantize_weight   the same over a [out, in] weight's channels
  adaln_quantize    flux_norm.adaln_modulate straight into 8-bit rows
  int8_linear       act(rows @ weight^T + bias),  act = none or GELU(tanh)
  int8_qkv          the joint Q/K/V projection of [text; image] rows with the heads' RMSNorm of Q and K and
                    the rotation in the same pass, written as the [B, N, H, 128] storage of each that the
                    attention kernels read (flux_inputs.qk_prep_pair takes 16-bit projections instead)
  adaln_quantize_pair, int8_linear_pair
                    two row sets (a double block's image and text streams) in one launch

The products are summed as whole numbers and what follows is fp32, rounded once to the 16-bit output; a
row that holds an infinity or a NaN gives NaN.  Inference only: inputs that need a gradient are refused.
Launches are asynchronous on the current stream, need no workspace and can be captured into a graph.
The reference runs these layers in 16 bits (in the transformer that hilberta/flux_adapter.py wraps).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops

HEAD_DIM = 128
MAX_FEATURES = 1 << 17  # a sum of so many products fits 32 bits


def padded_features(features):
    """Columns of 8-bit rows of ``features`` values: filled up with zeros to a multiple of 64."""
    return -(-features // 64) * 64


class Int8Rows(NamedTuple):
    """Activations in 8 bits: q int8 [..., rows, padded_features(features)], zeros past ``features``, scale
    float32 [..., rows]; ``dtype`` is that of the 16-bit rows they stand for, and of products with them."""

    q: torch.Tensor
    scale: torch.Tensor
    features: int
    dtype: torch.dtype


class Int8Weight(NamedTuple):
    """A linear layer's weight in 8 bits: q int8 [out_features, padded_features(features)], zeros past
    ``features``, scale float32 [out_features]."""

    q: torch.Tensor
    scale: torch.Tensor
    features: int


def quantize_rows(x):
    """Int8Rows of 16-bit rows x [rows, features] or [B, rows, features] (contiguous last dimension)."""
    q, scale = ops.int8_rows(x)
    return Int8Rows(q, scale, x.shape[-1], x.dtype)


def quantize_weight(weight):
    """Int8Weight of a 16-bit weight [out_features, in_features]."""
    if weight.ndim != 2 or not weight.numel():
        raise ValueError("weight must be a nonempty [out_features, in_features] matrix")
    q, scale = ops.int8_rows(weight.detach())
    return Int8Weight(q, scale, weight.shape[1])


def adaln_quantize(x, shift, scale, *, y=None, gate=None, x_out=None, eps=1e-6):
    """Int8Rows of shift + LayerNorm(r) * (1 + scale), r = x + gate * y, in one pass; r is stored in
    ``x_out`` (which may be x) rounded, and normalised before that rounding.  Arguments as
    flux_norm.adaln_modulate's; hidden is any multiple of 8 up to 8192."""
    q, row_scale = ops.int8_adaln(x, shift, scale, y, gate, x_out, eps)
    return Int8Rows(q, row_scale, x.shape[-1], x.dtype)


def adaln_quantize_pair(first, second, *, eps=1e-6):
    """adaln_quantize of two row sets in one launch: ``first`` and ``second`` are its arguments as dicts, of
    one batch, hidden size, dtype and device; either may have no rows.  Returns both Int8Rows."""
    sets = [(s["x"], s["shift"], s["scale"], s.get("y"), s.get("gate"), s.get("x_out")) for s in (first, second)]
    q, scale, q2, scale2 = ops.int8_adaln_pair(*sets[0], *sets[1], eps)
    x, x2 = first["x"], second["x"]
    return Int8Rows(q, scale, x.shape[-1], x.dtype), Int8Rows(q2, scale2, x2.shape[-1], x2.dtype)


def _rows(x):
    return x if isinstance(x, Int8Rows) else quantize_rows(x)


def _check_features(weight, features):
    if weight.features != features:
        raise ValueError(f"the weight takes {weight.features} features, the rows have {features}")


def int8_linear(x, weight, bias=None, *, gelu=False, out=None):
    """act(x @ weight^T + bias) for x Int8Rows, or 16-bit rows that are quantized first, and an Int8Weight;
    act is GELU(tanh) with ``gelu``.  (A few 16-bit rows are quantized in the product's launch, to the same
    result.)  bias [out_features] in the rows' dtype.  ``out`` [..., rows,
    out_features] may be a row range or a column block of a larger buffer."""
    if out is not None:
        args, out = _linear(x, weight, bias, out)
        ops.int8_linear_out(*args, gelu)
        return out
    w, w_scale, features = weight
    if isinstance(x, Int8Rows):
        q, scale, n, dtype = x
        if n != features:
            _check_features(weight, n)
        return ops.int8_linear(q, scale, w, w_scale, bias, dtype, gelu)
    if x.shape[-1] != features:
        _check_features(weight, x.shape[-1])
    return ops.int8_linear_rows(x, w, w_scale, bias, gelu)


def _linear(x, weight, bias=None, out=None):
    """Arguments of one row set for the operators that write ``out``, and it."""
    q, scale, features, dtype = _rows(x)
    _check_features(weight, features)
    if out is None:
        out = torch.empty(*q.shape[:-1], weight.q.shape[0], dtype=dtype, device=q.device)
    elif out.dtype != dtype:
        raise ValueError("out must have the rows' dtype")
    return (q, scale, weight.q, weight.scale, bias, out), out


def int8_linear_pair(first, second, *, gelu=False):
    """int8_linear of two row sets in one launch: ``first`` and ``second`` are dicts of x, weight, bias and
    out, of one batch, layer shape, dtype and device; either may have no rows.  Returns both outputs."""
    a, out_a = _linear(**first)
    b, out_b = _linear(**second)
    ops.int8_linear_pair_out(*a, *b, gelu)
    return out_a, out_b


def int8_qkv(text, image, *, heads, weights, biases=(None, None), norms=((None, None), (None, None)), eps=1e-6,
             cos=None, sin=None, out=None):
    """[text; image] tokens -> out [3, B, T + n, heads, 128]: Q and K normalised and rotated, and V.

    ``text`` [B, T, features] (or None: T = 0) and ``image`` [B, n, features] are Int8Rows, or 16-bit rows
    that are quantized first; ``weights`` and ``biases`` = (text, image) are Int8Weights and biases of the
    columns [Q | K | V], heads * 128 each; ``norms`` = ((q_text, q_image), (k_text, k_image)) the RMSNorm
    weights [128] (None: no weight); cos/sin float32 [T + n, 128] in token order (None: no rotation)."""
    q, scale, features, dtype = _rows(image)
    (wt, wi), (bt, bi), ((qt, qi), (kt, ki)) = weights, biases, norms
    t = (None,) * 7
    if text is not None:
        text_q, text_scale, text_features, text_dtype = _rows(text)
        if text_features != features or text_dtype != dtype:
            raise ValueError("text and image rows must share features and dtype")
        if text_q.size(-2):
            t = (text_q, text_scale, wt.q, wt.scale, bt, qt, kt)
    if wi.features != features or (t[0] is not None and wt.features != features):
        raise ValueError("the weights must take the rows' features")
    if out is None:
        return ops.int8_qkv(*t, q, scale, wi.q, wi.scale, bi, qi, ki, cos, sin, dtype, heads, eps)
    if out.dtype != dtype:
        raise ValueError("out must have the rows' dtype")
    ops.int8_qkv_out(*t, q, scale, wi.q, wi.scale, bi, qi, ki, cos, sin, out, eps)
    return out
