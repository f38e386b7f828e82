"""How near the 8-bit blocks have to be to their plain form (oracle/int8_blocks.py), and data that shows each part.

Both forms round at the same places.  They differ where an fp32 value and its 64-bit one fall on two sides of a
rounding's border, and at the most as two independent roundings do, sqrt(2) of one.  A row rounded to whole steps
of its top / 127 is off by a step / sqrt(12), 1 % of itself for tops of 4.5 times the root mean square and 1.8 %
for 8 times (GELU's outputs); two such rows by 1.4 and 2.5 %.  In a block:

    V by its rows' 1.4 %; Q and K too, and the logits, sums of 128 products over sqrt(128) of values around 1, by
    2 x 1.4 % added in squares: 2.0 % of 1, which is the change of a weight of the softmax;
    attention's output by 1.4 and 2.0 %: 2.4;  its rows add 1.4: 2.8 % of the first update;
    the MLP's rows by as much and 1.4: 3.1, GELU's outputs by 2.5 more: 4.0 % of the second update;
    16-bit roundings by 2^-9 of the value each, well below.

So 5 % of an update, and of the rows that follow, which add 1.4 % to a share of that, and of Q, K and V as attention
is given them.
"""

import torch

BOUND = 0.05


def off(got, want):
    """Relative L2 distance."""
    got, want = got.double(), want.double()
    return float((got - want).norm() / want.norm())


class Attention:
    """The transformer's attention argument, as its formula in 64 bits; keeps the layers it was called for and what it
    was given, [B, N, heads, 128]."""

    layout = None

    def __init__(self):
        self.layers, self.given = [], []

    def __call__(self, layer, q, k, v, out):
        from oracle import int8_blocks as B

        self.layers.append(layer)
        self.given.append([t.transpose(1, 2).clone() for t in (q, k, v)])
        out.copy_(B.attend(*self.given[-1]).unflatten(-1, (-1, q.shape[-1])).transpose(1, 2))


def raise_parameters(w, gen):
    """A block's biases and head norms, in place, to sizes at which a missing or exchanged one shows."""
    def walk(value):
        if isinstance(value, torch.Tensor) and value.ndim == 1 and value.dtype in (torch.bfloat16, torch.float16):  # (no scale)
            yield value
        elif isinstance(value, (tuple, list)):
            for v in value:
                yield from walk(v)

    for name, value in w.items():
        for t in walk(value):
            mean, std = (1.0, 0.3) if name.startswith("norm") else (0.0, 0.5)
            t.copy_(mean + std * torch.randn(t.shape, generator=gen, device=gen.device))
