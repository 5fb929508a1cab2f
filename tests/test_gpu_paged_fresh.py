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


def test_captured_fresh_sequences_follow_their_inputs():
    """One graph of a batch with padding behind its sequences, replayed with other starts and positions, against the eager layer on a second pool."""
    torch.manual_seed(5)
    a, _ = block(torch.bfloat16)
    caches = [nv.PagedCache.new(16, KEY_HEADS, 16, DIM) for _ in range(2)]
    page_table = torch.randperm(16, device="cuda").to(torch.int32).reshape(2, 8)
    x = torch.randn(70, DIMS, device="cuda").bfloat16()
    positions, sequences, starts = ints([-1] * 70), ints([0] * 70), ints([0, 0, 0])
    rotary, ids, lengths = torch.zeros(3, 70, dtype=torch.int32, device="cuda"), ints([-1] * 70), ints([0, 0])
    run = lambda cache: a(x, cache, page_table, positions, lengths, sequences, starts, 70, rotary, ids, True)
    run(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(caches[0])
    for rows in ([40, 20], [1, 69], [0, 33], [70, 0], [5, 5]):
        n = sum(rows)
        x.normal_()
        positions.copy_(ints([*range(rows[0]), *range(rows[1]), *[-1] * (70 - n)]))
        sequences.copy_(ints([0] * rows[0] + [1] * (70 - rows[0])))
        starts.copy_(ints([0, rows[0], n]))
        rotary.copy_(torch.randint(0, 140, (3, 70)).to(torch.int32))  # (some outside the table of 128)
        ids.copy_((torch.arange(70) % 4 - 1).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = run(caches[1])
        assert torch.equal(y[:n], want[:n])
        for one, other in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
            assert torch.equal(one.weight.view(torch.int32), other.weight.view(torch.int32)) and torch.equal(one.scales, other.scales)
