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
