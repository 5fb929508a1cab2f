"""Scores of any finite size: a row that sees keys is never taken for one that sees none."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY, dense, random_cache
from tests.test_gpu_paged_attention import ints, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length,rows", [(5, 1), (2000, 1), (300, 90), (2000, 60)])
def test_low_scores(dtype, length, rows):
    """Equal keys, so equal weights, at scores of -6.4e31: the result is the mean of the values.  Equal scores have equal float32 errors, and a weight is 1
    (its product with a scale 16 bits, 24 in float32); 64 roundings of the sums, then the result's own."""
    torch.manual_seed(0)
    page_table, pages = tables([length], 16)
    cache = random_cache(pages, 2, 16, 64, nv.Quant.affine(32, 4), dtype)
    cache.keys.weight.view(torch.int32).fill_(0)
    cache.keys.scales.fill_(1.0)
    cache.keys.biases.fill_(1.0)
    q = torch.ones(rows, 8, 64, device="cuda", dtype=dtype)
    got = nv.paged_attention(q, cache, page_table, ints([length]), -1e30, ints([0, rows]), causal=False)
    v, _, size = dense(cache.values, page_table, 0, length)
    want = v.mean(1).repeat_interleave(4, 0)
    slack = (64 * 2.0 ** -24 + (2.0 ** -24 if dtype == torch.float32 else 2.0 ** -16)) * size.amax()
    assert ((got.double() - want).abs() <= HALF[dtype] * want.abs() + slack + TINY[dtype]).all()
    assert (nv.paged_attention(q, cache, page_table, ints([0]), -1e30, ints([0, rows]), causal=False) == 0).all()
