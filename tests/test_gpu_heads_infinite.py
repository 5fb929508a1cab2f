"""Infinities under the norm of a head: its finite values become zeros (x / sqrt(infinity)), the infinite ones NaN, other heads stay as they are."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY, normed, table, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,dims", [(128, 0), (128, 64), (128, 50), (64, 64), (80, 38), (320, 64)])
def test_an_infinite_value(dtype, dim, dims):
    """Two infinities in one head of three, a NaN in another; bounds as those of finite heads (three roundings of the norm's in float32, three of the
    rotation's, then the result's)."""
    torch.manual_seed(dim + dims)
    rotation = nv.Rotation(table(20, dims)) if dims else None
    x = torch.randn(2, 3, 5, dim, device="cuda").to(dtype)
    x[0, 1, :, 7], x[0, 1, :, dim - 1], x[1, 2, 3, 0] = float("inf"), -float("inf"), float("nan")
    w = (1 + 0.1 * torch.randn(dim, device="cuda")).to(dtype)
    want = size = normed(x, w, 1e-6)
    if rotation:
        want, size = turned(want, rotation.table[:5], False)
    for got in nv.head_norm_rope(x, x, w, w, rotation):
        assert torch.equal(got.isnan(), want.isnan()) and (got[0, 1].nan_to_num(0.0) == 0).all()
        u, slack = HALF[dtype], (8 * 2.0 ** -24 * size.abs()).nan_to_num(0.0)
        assert ((got.double() - want).nan_to_num(0.0).abs() <= u * (want.nan_to_num(0.0).abs() + slack) + slack + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_an_infinite_key(dtype):
    """The groups of the cache around it hold zeros, where they held NaN scales."""
    cache = nv.PagedCache.new(1, 1, 16, 128, nv.Quant.affine(32, 8), dtype)
    k, w = torch.randn(3, 1, 128, device="cuda").to(dtype), torch.ones(128, device="cuda", dtype=dtype)
    k[1, 0, 40] = float("inf")
    at = torch.arange(3, dtype=torch.int32, device="cuda")
    table0 = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    nv.append_paged(cache, k, k.nan_to_num(posinf=0.0), table0, at, torch.zeros_like(at), k_weight=w)
    keys, _ = nv.read_paged(cache, table0, at, torch.zeros_like(at))
    assert (keys[1] == 0).all() and keys.isfinite().all() and (keys[0] != 0).any()
