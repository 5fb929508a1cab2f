"""`layers.PagedAttention`: prompts and steps of several sequences through one pool."""
import pytest
import torch

import nuvec_amd as nv
from nuvec_amd.layers import PagedAttention, QuantizedLinear
from tests.paged_reference import attention

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def layer(dims, heads, key_heads, dim, norms, dtype, **more):
    put = lambda n, k: QuantizedLinear.from_linear((torch.randn(n, k, device="cuda") * k ** -0.5).to(dtype))
    weight = lambda: (1 + 0.1 * torch.randn(dim, device="cuda")).to(dtype) if norms else None
    return PagedAttention(put(heads * dim, dims), put(key_heads * dim, dims), put(key_heads * dim, dims), put(dims, heads * dim), heads, key_heads,
                          nv.Rotation.new(dim, 128), weight(), weight(), **more)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norms,window", [(False, 0), (True, 9)])
def test_prompts_and_steps(dtype, norms, window):
    """The operators' composition, bit for bit; their attention against 64 bits over what the cache holds."""
    torch.manual_seed(1)
    dims, heads, key_heads, dim, page = 256, 4, 2, 64, 16
    a = layer(dims, heads, key_heads, dim, norms, dtype, sinks=torch.randn(heads, device="cuda").to(dtype), window=window)
    caches = [nv.PagedCache.new(16, key_heads, page, dim, nv.Quant.affine(32, 8), dtype) for _ in range(2)]
    page_table = torch.randperm(16, device="cuda").to(torch.int32).reshape(2, 8)
    lengths = [0, 0]
    for rows in ([40, 3], [1, 1], [1, 60], [1, 1]):
        n = sum(rows)
        x = torch.randn(n, dims, device="cuda").to(dtype)
        positions = ints([*range(lengths[0], lengths[0] + rows[0]), *range(lengths[1], lengths[1] + rows[1])])
        lengths = [i + j for i, j in zip(lengths, rows)]
        step = n == 2
        sequences, starts = (None, None) if step else (ints([0] * rows[0] + [1] * rows[1]), ints([0, rows[0], n]))
        got = a(x, caches[0], page_table, positions, ints(lengths), sequences, starts, None if step else max(rows))
        q, k, v = (p(x).view(n, -1, dim) for p in (a.q_proj, a.k_proj, a.v_proj))
        q = nv.append_paged(caches[1], k, v, page_table, positions, sequences, a.rotation, a.k_norm, q, a.q_norm)
        y = nv.paged_attention(q, caches[1], page_table, ints(lengths), dim ** -0.5, starts, None if step else max(rows), a.sinks, window=window)
        assert got.shape == x.shape and torch.equal(got, a.o_proj(y.flatten(1)))
        want, bound = attention(q, caches[0], page_table, lengths, dim ** -0.5, None if step else [0, rows[0], n], a.sinks, window=window)
        assert ((y.double() - want).abs() <= bound).all()


def test_what_it_refuses():
    a = layer(128, 2, 1, 64, False, torch.bfloat16)
    cache, x, table = nv.PagedCache.new(2, 1, 16, 64), torch.zeros(1, 128, device="cuda", dtype=torch.bfloat16), ints([[0, 1]])
    with pytest.raises(nv.InvalidArgument, match="go together"):
        a(x, cache, table, ints([0]), ints([1]), sequences=ints([0]))
    with pytest.raises(nv.InvalidArgument, match="tokens must be"):
        a(x[None], cache, table, ints([0]), ints([1]))
    a.query_heads = 3
    with pytest.raises(nv.InvalidArgument, match="128 projected values of 3 heads"):
        a(x, cache, table, ints([0]), ints([1]))


def test_captured_steps_follow_their_inputs():
    """One graph of a decode step, replayed over growing sequences, against the eager layer on a second pool."""
    torch.manual_seed(3)
    a = layer(128, 4, 2, 64, True, torch.bfloat16)
    caches = [nv.PagedCache.new(8, 2, 16, 64) for _ in range(2)]
    table = ints([[3, 1, 0, 2], [4, 7, 6, 5]])
    x, positions, lengths = torch.randn(2, 128, device="cuda", dtype=torch.bfloat16), ints([-1, -1]), ints([0, 0])
    a(x, caches[0], table, positions, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a(x, caches[0], table, positions, lengths)
    for step in range(20):
        x.normal_()
        positions.copy_(ints([step, 2 * step]))
        if step == 7:
            positions[1] = -1  # (padding: nothing is written)
        lengths.copy_(ints([step + 1, 2 * step + 1]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, a(x, caches[1], table, positions, lengths)), step
    for one, other in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
        assert torch.equal(one.weight.view(torch.int32), other.weight.view(torch.int32)) and torch.equal(one.scales, other.scales)


def test_captured_batches_follow_their_inputs():
    """One graph of 64 rows for prompts, steps and padding, whose starts, positions and lengths change between the replays; padding rows' keys are
    not written, and the others' results are those of a call without them."""
    torch.manual_seed(4)
    a = layer(128, 4, 2, 64, True, torch.bfloat16)
    caches = [nv.PagedCache.new(24, 2, 16, 64) for _ in range(2)]
    table = torch.randperm(24, device="cuda").to(torch.int32).reshape(2, 12)
    x = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16)
    positions, sequences, starts, lengths = ints([-1] * 64), ints([0] * 64), ints([0, 0, 0]), ints([0, 0])
    a(x, caches[0], table, positions, lengths, sequences, starts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a(x, caches[0], table, positions, lengths, sequences, starts)
    held = [0, 0]
    for rows in ([60, 4], [1, 1], [1, 50], [0, 3], [20, 20]):
        n = sum(rows)
        x.normal_()
        now = [h + r for h, r in zip(held, rows)]
        positions.copy_(ints([*range(held[0], now[0]), *range(held[1], now[1])] + [-1] * (64 - n)))
        sequences.copy_(ints([0] * rows[0] + [1] * rows[1] + [0] * (64 - n)))
        starts.copy_(ints([0, rows[0], n]))
        lengths.copy_(ints(now))
        held = now
        graph.replay()
        torch.cuda.synchronize()
        eager = a(x, caches[1], table, positions, lengths, sequences, starts)
        assert torch.equal(y[:n], eager[:n]), rows
        for one, other in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
            assert torch.equal(one.weight.view(torch.int32), other.weight.view(torch.int32)) and torch.equal(one.scales, other.scales) and torch.equal(one.biases, other.biases)
    assert held == [82, 78]


def test_no_tokens():
    a = layer(128, 2, 1, 64, False, torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    y = a(torch.zeros(0, 128, device="cuda", dtype=torch.bfloat16), nv.PagedCache.new(2, 1, 16, 64), ints([[0, 1]]), none, ints([0]), none, ints([0, 0]))
    assert y.shape == (0, 128)
