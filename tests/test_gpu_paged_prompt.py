"""Attention of many lines over a paged cache (csrc/paged_prompt_kernel.h): block and tile edges, splits that see nothing, mixtures with few lines."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import attention, random_cache
from tests.test_gpu_paged_attention import check, ints, tables

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rep,rows", [(1, 49), (4, 12), (4, 13), (1, 127), (1, 128), (1, 129), (3, 43), (7, 19), (8, 31), (8, 33), (5, 77), (64, 3)])
def test_lines_at_the_edges_of_blocks(dtype, rep, rows):
    """Alone, and beside a sequence of one row; on the diagonal, behind a prefix, more rows than positions."""
    for length in (rows, rows + 45, rows - 1, 1):
        check(64, 32, 4, dtype, rep, 1, 16, [length], [rows])
    check(128, 64, 8, dtype, rep, 2, 64, [rows + 100, 70, 0, rows], [rows, 1, 0, rows], sinks=True)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,group,bits", [(128, 64, 4), (128, 32, 8), (128, 128, 4), (64, 64, 8), (64, 32, 4)])
def test_splits_that_see_nothing(dtype, dim, group, bits):
    """Long prompts on the diagonal, whose first rows see none of the later splits' positions; behind a long prefix; a window that leaves most
    splits out; every position seen."""
    check(dim, group, bits, dtype, 4, 1, 64, [1500], [1500])
    check(dim, group, bits, dtype, 4, 2, 128, [4000], [70])
    check(dim, group, bits, dtype, 2, 1, 32, [3000], [400], window=50, sinks=True)
    check(dim, group, bits, dtype, 2, 1, 32, [3000, 800], [40, 300], causal=False)
    check(dim, group, bits, dtype, 2, 1, 32, [600, 3], [900, 80])  # (300 rows of the first and 77 of the second see nothing)


@pytest.mark.parametrize("dtype", HALVES)
def test_mixtures(dtype):
    """More sequences than a wavefront has lanes, prompts among single tokens; sized for one row and for more."""
    g = torch.Generator().manual_seed(4)
    rows = torch.randint(0, 4, (70,), generator=g).tolist()
    lengths = [n + int(torch.randint(0, 300, (1,), generator=g)) for n in rows]
    rows[5], lengths[5], rows[40], lengths[40], rows[69], lengths[69] = 200, 900, 33, 33, 65, 2000
    for hint in (1, 65, None):
        check(128, 64, 4, dtype, 4, 2, 64, lengths, rows, hint=hint)


def test_one_sequence_shorter_than_its_call():
    """A call sized for many lines of one sequence that has few, or none: rows behind its end stay as they were."""
    page_table, pages = tables([300], 64)
    cache = random_cache(pages, 2, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    q = torch.randn(40, 8, 128, device="cuda", dtype=torch.bfloat16)
    for rows in (0, 1, 3, 40):
        out = torch.full_like(q, 7.0)
        nv.paged_attention(q, cache, page_table, ints([300]), 0.1, ints([0, rows]), out=out)
        want, bound = attention(q, cache, page_table, [300], 0.1, [0, rows])
        assert ((out.double() - want).abs() <= bound)[:rows].all() and (out[rows:] == 7).all(), rows


def test_captured_prompts_follow_their_lengths():
    """Two graphs of one shape over prompts that move between the rows, from one split to several, other work between the replays."""
    torch.manual_seed(6)
    page_table, pages = tables([4096, 4096], 64)
    cache = random_cache(pages, 2, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    q = torch.randn(260, 8, 128, device="cuda", dtype=torch.bfloat16)
    lengths, starts = ints([1, 9]), ints([0, 1, 2])
    run = lambda out: nv.paged_attention(q, cache, page_table, lengths, 0.1, starts, out=out)
    outs = [torch.zeros_like(q) for _ in range(3)]
    run(outs[2])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            run(out)
    for a, b, at, end in ((300, 40, 200, 240), (4096, 4096, 1, 260), (256, 4000, 0, 255), (33, 2, 33, 35), (4096, 0, 260, 260)):
        lengths.copy_(ints([a, b]))
        starts.copy_(ints([0, at, end]))
        q.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        run(outs[2])
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]), (a, b)
        want, bound = attention(q, cache, page_table, [a, b], 0.1, [0, at, end])
        assert ((outs[2].double() - want).abs() <= bound)[:end].all()


def test_prompts_on_two_streams_at_once():
    page_table, pages = tables([3000, 2000], 64)
    cache = random_cache(pages, 4, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    qs = [torch.randn(150, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    lengths, starts = ints([3000, 2000]), ints([0, 149, 150])
    want = [nv.paged_attention(q, cache, page_table, lengths, 0.1, starts) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(nv.paged_attention(qs[i], cache, page_table, lengths, 0.1, starts))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("bits", [4, 8])
def test_pages_beyond_32_bits(bits):
    """Pages at the end of a pool whose codes are more than 2^32 bytes, beside its first."""
    pages = (1 << 32) // (8 * 1024 * 128 * bits // 8) + 2
    empty = lambda last, t: torch.empty((pages, 8, 1024, last), dtype=t, device="cuda")
    of = lambda: nv.Quantized.affine(empty(4 * bits, torch.int32).view(torch.uint32), empty(2, torch.float16), empty(2, torch.float16), 64, bits)
    cache = nv.PagedCache(of(), of())
    page_table = ints([[pages - 1, 0, pages - 2]])
    torch.manual_seed(0)
    k, v = (torch.randn(2100, 8, 128, device="cuda", dtype=torch.float16) for _ in range(2))
    nv.append_paged(cache, k, v, page_table, ints(range(2100)), torch.zeros(2100, dtype=torch.int32, device="cuda"))
    q = torch.randn(40, 16, 128, device="cuda", dtype=torch.float16)
    got = nv.paged_attention(q, cache, page_table, ints([2100]), 0.1, ints([0, 40]))
    want, bound = attention(q, cache, page_table, [2100], 0.1, [0, 40])
    assert ((got.double() - want).abs() <= bound).all()


def test_calls_of_nothing():
    """No rows, no lengths, sequences without rows around one that has some."""
    page_table, pages = tables([300, 300, 300], 64)
    cache = random_cache(pages, 2, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    q = torch.randn(40, 8, 128, device="cuda", dtype=torch.bfloat16)
    assert nv.paged_attention(q[:0], cache, page_table, ints([300, 300, 300]), 0.1, ints([0, 0, 0, 0])).shape == (0, 8, 128)
    out = torch.full_like(q, 7.0)
    nv.paged_attention(q, cache, page_table, ints([300, 300, 300]), 0.1, ints([0, 0, 0, 0]), out=out)
    assert (out == 7).all()
    nv.paged_attention(q, cache, page_table, ints([0, 0, 0]), 0.1, ints([0, 0, 40, 40]), out=out)
    assert (out == 0).all()
