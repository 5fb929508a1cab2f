"""Calls of `PagedAttention` that are refused before anything is computed.  No GPU."""
import pytest
import torch

import nuvec_amd as nv
from nuvec_amd.layers import PagedAttention, QuantizedLinear

ints = lambda *s: torch.zeros(s, dtype=torch.int32)


@pytest.mark.parametrize("fresh", [False, True])
def test_rotary_positions_need_a_rotation(fresh):
    linear = QuantizedLinear(torch.zeros(64, 8, dtype=torch.uint32), torch.zeros(64, 1), torch.zeros(64, 1), None, nv.Quant.affine(64, 4))
    layer = PagedAttention(linear, linear, linear, linear, 1, 1)
    with pytest.raises(nv.InvalidArgument, match="without a rotation"):
        layer(torch.zeros(2, 64), nv.PagedCache.new(2, 1, 16, 64, device="cpu"), ints(1, 2), ints(2), ints(1), ints(2), ints(2), 2, ints(2), fresh=fresh)
