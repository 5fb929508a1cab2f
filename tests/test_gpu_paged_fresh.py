"""`PagedAttention` of fresh sequences writes the cache where the same call over the cache does."""
import pytest
import torch

import nuvec_amd as nv
from nuvec_amd import layers
from tests.test_gpu_serving_block import DIM, DIMS, KEY_HEADS, block, ints

pytestmark = pytest.mark.gpu


def rows_written(a, x, page_table, args, more):
    """Whether the keys of each place of the cache are written, by a pool of codes that no key has."""
    cache = nv.PagedCache.new(16, KEY_HEADS, 16, DIM, nv.Quant.affine(32, 8), x.dtype)
    for t in (cache.keys, cache.values):
        t.scales.fill_(float("nan"))
    a(x, cache, page_table, *args, **more)
    return [(~t.scales.isnan()).all(-1) for t in (cache.keys, cache.values)]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_positions_outside_the_table_write_nothing(dtype, native, monkeypatch):
    """One token's position, or one axis's, at the end of the table or beyond it, or negative."""
    if not native:  # (the package's own checks and calls)
        class Declines:
            def __getattr__(self, name):
                return lambda *args: None
        monkeypatch.setattr(nv._lib, "_native", Declines())
    torch.manual_seed(3)
    a, _ = block(dtype)
    a.rotation = nv.Rotation.new(DIM, 30, axes=a.rotation.axes)
    plain = layers.PagedAttention(*(getattr(a, n) for n in ("q_proj", "k_proj", "v_proj", "o_proj", "query_heads", "key_heads")), nv.Rotation.new(DIM, 30))
    bare = layers.PagedAttention(*(getattr(a, n) for n in ("q_proj", "k_proj", "v_proj", "o_proj", "query_heads", "key_heads")))
    page_table = torch.randperm(16, device="cuda").to(torch.int32).reshape(2, 8)
    x = torch.randn(60, DIMS, device="cuda").to(dtype)
    positions = ints([*range(40), *range(20)])  # (the last ten of the first sequence lie outside the table)
    positions[50] = -1
    args = (positions, ints([40, 20]), ints([0] * 40 + [1] * 20), ints([0, 40, 60]), 40)
    one, several = positions.clamp(0, 29), positions.clamp(0, 29).repeat(3, 1)
    one[3], one[7], one[45] = 30, -1, 1 << 30
    several[0, 3], several[1, 7], several[2, 45], several[1, 46] = 30, -1, 1 << 30, 29
    for layer, rotary in ((a, None), (a, one), (a, several), (plain, None), (plain, one), (bare, None)):
        fresh, other = (rows_written(layer, x, page_table, args, {"rotary_positions": rotary, "fresh": f}) for f in (True, False))
        assert all(torch.equal(f, o) for f, o in zip(fresh, other))
        missing = {None: 11, 1: 4, 2: 4}[None if rotary is None else rotary.ndim] if layer is not bare else 1
        assert fresh[0].sum().item() == (60 - missing) * KEY_HEADS
