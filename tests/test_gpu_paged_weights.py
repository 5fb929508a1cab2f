"""The softmax's weights in attention over a paged cache hold 16 bits in bfloat16, so that the result is off by its own rounding alone."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, dense, random_cache
from tests.test_gpu_paged_attention import ints, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,group,bits", [(128, 64, 4), (128, 32, 4), (128, 128, 8), (64, 64, 8), (64, 32, 4)])
@pytest.mark.parametrize("length,rows", [(9, 1), (40, 3), (700, 1), (300, 150)])
def test_weights_of_16_bits(dim, group, bits, length, rows):
    """Values of both signs, nearly even weights: results are small beside the values, and so is their rounding beside one of the weights to 8 bits.

    The bound: a weight x scale in two terms of bfloat16 is off by 2^-16 of itself, and multiplies operands of at most 2^(bits + 1).  Scores are
    float32 sums of the products of 64 or 128 values and their biases, 32 roundings of 2^-24 of the sum of their sizes; an error e of theirs moves
    the result by at most 2 e max |v|.  The weighted sums likewise 64 roundings of the values' sizes, then the result's own."""
    torch.manual_seed(dim + length)
    heads, scale = 8, dim ** -0.5
    page_table, pages = tables([length], 16)
    cache = random_cache(pages, 1, 16, dim, nv.Quant.affine(group, bits), torch.bfloat16)
    q = (0.1 * torch.randn(rows, heads, dim, device="cuda")).bfloat16()
    got = nv.paged_attention(q, cache, page_table, ints([length]), scale, ints([0, rows])).double().transpose(0, 1)  # [heads, rows, dim]
    k, _, k_size = dense(cache.keys, page_table, 0, length)
    v, _, v_size = dense(cache.values, page_table, 0, length)
    x = q.double().transpose(0, 1)
    hidden = torch.arange(length, device="cuda") > (length - rows + torch.arange(rows, device="cuda"))[:, None]
    p = torch.softmax((scale * x @ k.transpose(1, 2)).masked_fill(hidden, float("-inf")), -1)
    e = 32 * 2.0 ** -24 * scale * (x.abs() @ k_size.transpose(1, 2)).amax(-1, keepdim=True)
    slack = 2 * e * v.abs().max() + 64 * 2.0 ** -24 * v_size.max()
    want = p @ v
    off = (got - want).abs() - HALF[torch.bfloat16] * want.abs()
    assert (off <= 2.0 ** -16 * (p @ v_size) + slack).all(), off.max().item()
