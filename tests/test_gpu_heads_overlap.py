"""Rotary positions and norms of heads whose rows overlap in memory: results with rows of their own, those of a copy."""
import numpy as np
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import table

pytestmark = pytest.mark.gpu


def views(dtype):
    """Sliding windows, fewer than a head has values and more; every dimension one value apart; a single position of several heads."""
    x = torch.randn(1, 2, 330, device="cuda").to(dtype)
    yield x[..., :136].unfold(-1, 64, 1)
    yield x.unfold(-1, 64, 1)
    yield x[0, 0].as_strided((2, 3, 5, 64), (7, 1, 1, 1))
    yield x[0, 0].as_strided((1, 3, 1, 64), (1, 1, 1, 1))
    yield x[0, 0].as_strided((3, 2, 4, 64), (1, 64, 16, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_overlapping_rows(dtype):
    torch.manual_seed(0)
    rotation = nv.Rotation(table(300, 64))
    w = (1 + 0.1 * torch.randn(64, device="cuda")).to(dtype)
    for x in views(dtype):
        for offset in (3, np.int64(3)):  # (the second by way of the Python layer's own checks)
            y, want = nv.rope(x, rotation, offset), nv.rope(x.contiguous(), rotation, offset)
            assert y.stride(3) == 1 and torch.equal(y, want), x.stride()
            for one, other in zip(nv.head_norm_rope(x, x, w, None, rotation, offset), nv.head_norm_rope(x.contiguous(), x.contiguous(), w, None, rotation, offset)):
                assert one.stride(3) == 1 and torch.equal(one, other), x.stride()


def test_expanded_outputs_are_refused():
    """On the device too, where a call takes the native path first; a single row may have any stride."""
    rotation = nv.Rotation(table(300, 64))
    x = torch.randn(1, 1, 5, 64, device="cuda")
    wide = x.expand(2, 3, 5, 64)
    with pytest.raises(nv.InvalidArgument, match="share their memory"):
        nv.rope(wide, rotation, 3, out=wide)
    y = torch.zeros(330, device="cuda").as_strided((1, 1, 5, 64), (0, 0, 64, 1))
    assert nv.rope(x, rotation, 3, out=y) is y and torch.equal(y, nv.rope(x, rotation, 3))
