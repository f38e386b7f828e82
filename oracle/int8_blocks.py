"""A transformer's blocks with their linear layers in 8 bits, from their formulas in 64 bits.

What a block holds in 16 or in 8 bits is rounded here too: the heads of Q, K and V, attention's output, each linear
layer's output and the residual to 16, the rows of every linear layer to 8 with one scale a row.  Weights are
(q [columns, padded], scale [columns], features) with a bias; rows that enter or leave a block in 8 bits are the
values they stand for.

    double:  [q | k | v] of the text and image rows by weights of their own, one attention over [text; image]
             x += gate out(attention);   x += gate2 ff2(GELU(ff1(shift2 + LayerNorm(x) (1 + scale2))))
    single:  one weight for all rows;    x += gate out([attention | GELU(mlp(xn))])
and the rows that the next block reads, shift' + LayerNorm(x) (1 + scale').
"""

import math

import torch

from . import int8_ops as O


def attend(q, k, v):
    """Softmax attention of [B, N, heads, 128] heads, in 64 bits: [B, N, heads * 128]."""
    q, k, v = (t.double().transpose(1, 2).contiguous() for t in (q, k, v))
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    return torch.matmul(s.softmax(-1), v).transpose(1, 2).flatten(2)


def gelu(v):
    return O.gelu(v, torch.zeros_like(v))[0]


def held8(v):
    """What 8-bit rows of the values v stand for."""
    q, scale, _ = O.quantize(v)
    return q.double() * scale[..., None]


def _layer(v, weight, bias):
    q, scale, features = weight
    w = q[:, :features].double() * scale.double()[:, None]
    return (v.flatten(0, -2) @ w.t()).unflatten(0, v.shape[:-1]) + bias.double()


def _joint(layers, norms, rows, heads, cos, sin, eps, dtype):
    """Q, K and V [B, N, heads, 128] of the row sets one after another, rounded."""
    p = torch.cat([_layer(v, *layer) for v, layer in zip(rows, layers)], 1)
    q, k = (torch.cat([n.expand(v.shape[1], -1) for v, n in zip(rows, pair)]) for pair in norms)
    return [t.to(dtype) for t, _ in O.qkv(p, torch.zeros_like(p), heads, q, k, cos, sin, eps)]


def double_block(w, mods, x, xn, c, cn, cos, sin, next_mods, heads, eps=1e-6, attend=attend, act=gelu):
    """(x, xn, c, cn) after the block: residual streams x (image) and c (text) rounded to their type, xn and cn the
    8-bit rows that follow.  ``mods`` = (image's, text's) (shift, scale, gate, shift2, scale2, gate2), ``next_mods``
    their (shift, scale) after it."""
    T, dtype = c.shape[1], x.dtype
    o = attend(*_joint((w["qkv_c"], w["qkv_x"]), ((w["norm_added_q"], w["norm_q"]), (w["norm_added_k"], w["norm_k"])),
                       (cn, xn), heads, cos, sin, eps, dtype)).to(dtype)
    done = []
    for rows, part, (_, _, gate, shift, scale, gate2), following, s in ((x, o[:, T:], mods[0], next_mods[0], "x"),
                                                                       (c, o[:, :T], mods[1], next_mods[1], "c")):
        a = _layer(held8(part), *w["out_" + s]).to(dtype)
        m, _, r, _ = O.adaln(rows, shift, scale, a, gate, eps)
        first, second = w["ff_" + s]
        f = act(_layer(held8(m), *first)).to(dtype)
        f = _layer(held8(f), *second).to(dtype)
        m, _, r, _ = O.adaln(r.to(dtype), *following, f, gate2, eps)
        done += [r.to(dtype), held8(m)]
    return done


def single_block(w, mods, h, hn, T, cos, sin, next_mods, heads, eps=1e-6, attend=attend, act=gelu):
    """(h, m) after the block, for joint rows: the residual rounded to its type, and shift' + LayerNorm (1 + scale')
    of it before any rounding."""
    dtype = h.dtype
    o = attend(*_joint((w["qkv"],), ((w["norm_q"],), (w["norm_k"],)), (hn,), heads, cos, sin, eps, dtype)).to(dtype)
    both = torch.cat([o, act(_layer(hn, *w["mlp"])).to(dtype)], -1)
    m, _, r, _ = O.adaln(h, *next_mods, _layer(held8(both), *w["out"]).to(dtype), mods[2], eps)
    return r.to(dtype), m
