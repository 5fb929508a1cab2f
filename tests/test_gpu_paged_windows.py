"""Windows beyond every position are no window at all, however large the number."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import random_cache
from tests.test_gpu_paged_attention import ints, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [1 << 30, 1 << 31, (1 << 32) + 5, (1 << 63) - 1, (1 << 64) + 5])
@pytest.mark.parametrize("length,rows", [(20, 3), (20, 40), (300, 400), (300, 20), (700, 1)])
def test_windows_that_see_everything(window, length, rows):
    """Fewer rows than positions and more, on both kernels."""
    torch.manual_seed(length)
    page_table, pages = tables([length], 16)
    cache = random_cache(pages, 1, 16, 64, nv.Quant.affine(32, 4), torch.bfloat16)
    q = torch.randn(rows, 4, 64, device="cuda", dtype=torch.bfloat16)
    of = lambda window: nv.paged_attention(q, cache, page_table, ints([length]), 0.125, ints([0, rows]), window=window)
    assert torch.equal(of(window), of(0))
