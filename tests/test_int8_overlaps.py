"""What the 8-bit operators write lies apart from everything that a launch reads, the other set's operands among
it: other waves read those while it is written.

The operators make these checks on any device and refuse CPU tensors last, so each is seen here without a GPU:
a call that passes every check ends with that refusal.
"""

import pytest
import torch

from hilberta_amd import flux_int8 as f

BF16 = torch.bfloat16
ON_DEVICE = "device tensors"


def _refused(match, call, *args, **kwargs):
    with pytest.raises(ValueError, match=match):
        call(*args, **kwargs)


@pytest.mark.parametrize("writer", [0, 1])
@pytest.mark.parametrize("read", ["shift", "scale", "gate"])
def test_adaln_residual_over_the_other_sets_vectors(writer, read):
    B, C = 2, 64
    sets = [dict(x=torch.zeros(B, n, C, dtype=BF16), y=torch.zeros(B, n, C, dtype=BF16), x_out=torch.zeros(B, n, C, dtype=BF16),
                 **{k: torch.zeros(B, C, dtype=BF16) for k in ("shift", "scale", "gate")}) for n in (3, 5)]
    _refused(ON_DEVICE, f.adaln_quantize_pair, *sets)
    rows = sets[writer]["x_out"]
    over = rows.view(-1, C)[1:1 + B]  # rows 1 and 2 of what this set writes
    if read != "gate":  # (both share one batch stride, as these do)
        assert over.stride(0) == C
    sets[1 - writer][read] = over
    _refused("cannot alias", f.adaln_quantize_pair, *sets)
    sets[1 - writer][read] = torch.zeros(B, C, dtype=BF16)
    _refused(ON_DEVICE, f.adaln_quantize_pair, *sets)


@pytest.mark.parametrize("which", ["text_norm_q", "text_norm_k", "norm_q", "norm_k"])
def test_qkv_output_over_a_heads_norm(which):
    B, T, n, H = 2, 3, 5, 2
    rows = lambda k: f.Int8Rows(torch.zeros(B, k, 128, dtype=torch.int8), torch.zeros(B, k), 70, BF16)  # noqa: E731
    w = f.Int8Weight(torch.zeros(3 * H * 128, 128, dtype=torch.int8), torch.zeros(3 * H * 128), 70)
    out = torch.zeros(3, B, T + n, H, 128, dtype=BF16)
    norms = {k: torch.zeros(128, dtype=BF16) for k in ("text_norm_q", "text_norm_k", "norm_q", "norm_k")}

    def call(match):
        _refused(match, f.int8_qkv, rows(T), rows(n), heads=H, weights=(w, w), out=out,
                 norms=((norms["text_norm_q"], norms["norm_q"]), (norms["text_norm_k"], norms["norm_k"])))

    call(ON_DEVICE)
    norms[which] = out[1, 1, 4, 1]
    call("cannot alias")
