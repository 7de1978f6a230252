"""Calls at the edge of what the branch norms, the rotary positions with several axes, the moves of pages and the log probabilities
take, and the paths of models, pool, engine and server around them (CPU)."""
import struct

import pytest
import torch

from mlxcel_b200.ops import KVLayer, _lib, rotary


# ----------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("heads", [dict(Hq=0, Hkv=0), dict(Hq=2, Hkv=-1), dict(Hq=-2, Hkv=1), dict(Hq=1, Hkv=1, D=0)])
def test_mrope_append_refuses_a_projection_without_heads(heads):
    kw = dict(D=64) | heads
    hkv, D = max(kw["Hkv"], 0), kw["D"]
    slab = lambda: torch.zeros(4, hkv, 8, D)    # noqa: E731
    with pytest.raises(ValueError):
        rotary.mrope_append(torch.zeros(5, max(0, (kw["Hq"] + 2 * kw["Hkv"]) * D)), torch.zeros(3, 5, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                            torch.ones(0), torch.zeros(0, dtype=torch.int32), KVLayer(slab(), slab(), None, None, 8), rot_dim=0, **kw)


def test_mrope_entry_refuses_no_heads_before_it_launches():
    """The C entry checks this itself (it returns before it asks for a device)."""
    args = rotary._ARGS.pack(*([16, 0] * 3), 16, 16, 64, *[16] * 5, 0, 0, 3, 5, 0, 0, 64, 64, 16, 0, 16, 1e-6, 1.0)
    assert len(args) == struct.calcsize(rotary._ARGS.format) and _lib.load().mx_mrope_append(args, None) == -1
