"""Attention over a paged cache (csrc/paged_rows_kernel.h) against 64 bits; tests/paged_reference.py derives the bound."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import attention, random_cache

pytestmark = pytest.mark.gpu
FORMS = [(128, 64, 4), (128, 32, 4), (128, 128, 4), (64, 64, 4), (64, 32, 4), (128, 64, 8), (128, 32, 8), (128, 128, 8), (64, 64, 8), (64, 32, 8)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables(lengths, page, spare=3, columns=None, seed=0):
    """Shuffled pages; the entries behind a sequence's pages name none."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(held) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lengths), columns or max(1, max(held))), 1 << 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    return table.cuda(), sum(held) + spare


def check(dim, group, bits, dtype, rep, key_heads, page, lengths, rows=None, sinks=False, causal=True, window=0, seed=0, hint=None):
    torch.manual_seed(seed)
    page_table, pages = tables(lengths, page, seed=seed)
    cache = random_cache(pages, key_heads, page, dim, nv.Quant.affine(group, bits), dtype, seed)
    starts = None if rows is None else [0] + torch.tensor(rows).cumsum(0).tolist()
    n = len(lengths) if rows is None else starts[-1]
    q = torch.randn(n, rep * key_heads, dim, device="cuda").to(dtype)
    s = torch.randn(rep * key_heads, device="cuda").to(dtype) if sinks else None
    scale = dim ** -0.5
    got = nv.paged_attention(q, cache, page_table, ints(lengths), scale, None if rows is None else ints(starts), hint, s, causal, window)
    want, bound = attention(q, cache, page_table, lengths, scale, starts, s, causal, window)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()
    return cache, page_table, q, got


@pytest.mark.parametrize("dim,group,bits", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row(dim, group, bits, dtype):
    """No position, one, tiles and pages full and not, several splits; query heads that fill an instruction's columns, that do not, and more."""
    lengths = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 700]
    for rep, key_heads, page, sinks in ((4, 2, 16, False), (1, 3, 64, True), (7, 1, 32, False), (20, 1, 128, True)):
        check(dim, group, bits, dtype, rep, key_heads, page, lengths, sinks=sinks)


@pytest.mark.parametrize("dim,group,bits", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_several_rows(dim, group, bits, dtype):
    """Ragged rows, more rows than positions (the first of them see nothing), sequences without rows or positions; masks."""
    lengths, rows = [33, 5, 0, 70, 2, 300, 17, 64], [1, 5, 2, 20, 4, 9, 0, 33]
    check(dim, group, bits, dtype, 4, 2, 16, lengths, rows)
    check(dim, group, bits, dtype, 3, 1, 64, lengths, rows, sinks=True, window=11, hint=2)  # (more rows than the call is sized for)
    check(dim, group, bits, dtype, 8, 1, 32, lengths, rows, causal=False, hint=33)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 31, 32, 100, 1000])
def test_windows(dtype, window):
    check(128, 64, 4, dtype, 4, 2, 32, [1, 32, 99, 1500], window=window)
    check(64, 32, 8, dtype, 2, 1, 16, [40, 700, 1500], [40, 3, 64], window=window, sinks=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_splits(dtype):
    """One long sequence beside short ones, and more sequences than a wavefront has lanes: every number of splits, merged."""
    check(128, 64, 4, dtype, 4, 1, 256, [20000, 1, 0, 300, 4000])
    check(64, 64, 8, dtype, 2, 1, 64, [20000], sinks=True)
    check(128, 64, 4, dtype, 2, 1, 64, [(i * 53) % 700 for i in range(150)])
    check(64, 32, 4, dtype, 4, 1, 64, [(i * 91) % 2000 for i in range(70)], [i % 4 for i in range(70)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_positions_may_hold_anything(dtype):
    """NaN and infinities behind the lengths, in pages of nobody, in front of windows, and at positions that the causal mask hides from
    some rows: the rows that do not see them have the bits that they have without them."""
    torch.manual_seed(1)
    for rows, window in (([1, 1], 0), ([30, 9], 0), ([2, 40], 20)):
        lengths, page = [45, 300], 32
        page_table, pages = tables(lengths, page)
        cache = random_cache(pages, 2, page, 128, nv.Quant.affine(64, 4), dtype)
        starts = [0, rows[0], sum(rows)]
        q = torch.randn(starts[-1], 8, 128, device="cuda").to(dtype)
        run = lambda: nv.paged_attention(q, cache, page_table, ints(lengths), 0.1, ints(starts), None, None, True, window)
        clean = run()
        used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lengths):
            first = max(0, n - rows[b] - window + 1) if window else 0
            for p in range(first, n):
                used[page_table[b, p // page].long(), p % page] = True
        poison = (~used)[:, None, :, None].expand_as(cache.keys.scales)
        for t, value in ((cache.keys.scales, "nan"), (cache.keys.biases, "inf"), (cache.values.scales, "-inf"), (cache.values.biases, "nan")):
            t[poison] = float(value)
        assert torch.equal(run(), clean)
        # the last position of each sequence: its last row alone sees it
        for b, n in enumerate(lengths):
            at = (page_table[b, (n - 1) // page].long(), slice(None), (n - 1) % page)
            cache.keys.scales[at], cache.values.biases[at] = float("nan"), float("inf")
        got = run()
        for b in range(2):
            assert torch.equal(got[starts[b]:starts[b + 1] - 1], clean[starts[b]:starts[b + 1] - 1]) and got[starts[b + 1] - 1].isnan().all()


def test_rows_of_no_sequence_are_left():
    cache, page_table, q, got = check(128, 64, 4, torch.bfloat16, 4, 2, 32, [50, 60], [3, 2])
    more = torch.cat([q, torch.full_like(q, float("nan"))])
    out = torch.full((10, 8, 256), 7.0, device="cuda", dtype=torch.bfloat16)
    view = out[..., :128]
    assert nv.paged_attention(more, cache, page_table, ints([50, 60]), 128 ** -0.5, ints([0, 3, 5]), out=view) is view
    assert torch.equal(view[:5], got) and (view[5:] == 7).all() and (out[..., 128:] == 7).all()
    # starts that reach behind the rows, or descend, take the rows that there are
    nv.paged_attention(more[:4], cache, page_table, ints([50, 60]), 128 ** -0.5, ints([0, 3, 1 << 30]))
    nv.paged_attention(more[:4], cache, page_table, ints([50, 60]), 128 ** -0.5, ints([3, 0, -5]))


def test_strides_and_shared_pages():
    """Queries as a projection of queries, keys and values leaves them; two sequences with the same first pages; lengths beyond the table."""
    torch.manual_seed(0)
    cache = random_cache(5, 2, 32, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    page_table = ints([[0, 1, 2], [0, 1, 3], [4, 4, 4]])
    lengths = [90, 70, 10]
    wide = torch.randn(3, 1537, device="cuda").to(torch.bfloat16)
    for q in (wide[:, :1024].unflatten(-1, (8, 128)), wide[:, 1:1025].unflatten(-1, (8, 128)), wide[:1, :1024].unflatten(-1, (8, 128)).expand(3, 8, 128)):
        got = nv.paged_attention(q, cache, page_table, ints(lengths), 0.1)
        want, bound = attention(q, cache, page_table, lengths, 0.1)
        assert ((got.double() - want).abs() <= bound).all()
    q = wide[:, :1024].unflatten(-1, (8, 128))
    assert torch.equal(nv.paged_attention(q, cache, page_table, ints([1000, 70, -4]), 0.1)[:2], nv.paged_attention(q, cache, page_table, ints([96, 70, 0]), 0.1)[:2])
    wider = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wider[:, 2:5] = page_table
    assert torch.equal(nv.paged_attention(q, cache, wider[:, 2:5], ints(lengths), 0.1), nv.paged_attention(q, cache, page_table, ints(lengths), 0.1))


@pytest.mark.parametrize("bits", [4, 8])
def test_offsets_beyond_32_bits(bits):
    """Pages at the end of a pool whose codes are more than 2^32 bytes."""
    pages = (1 << 32) // (8 * 1024 * 128 * bits // 8) + 3
    dim, page, heads = 128, 1024, 8
    empty = lambda last, t: torch.empty((pages, heads, page, last), dtype=t, device="cuda")
    of = lambda: nv.Quantized.affine(empty(dim * bits // 32, torch.int32).view(torch.uint32), empty(2, torch.bfloat16), empty(2, torch.bfloat16), 64, bits)
    cache = nv.PagedCache(of(), of())
    page_table = ints([[pages - 1, 0], [pages - 2, pages - 3]])
    torch.manual_seed(0)
    k, v = (torch.randn(2100, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    sequences = ints([0] * 1050 + [1] * 1050)
    positions = ints(list(range(1050)) * 2)
    nv.append_paged(cache, k, v, page_table, positions, sequences)
    keys, values = nv.read_paged(cache, page_table, positions, sequences)
    for got, x in ((keys, k), (values, v)):
        assert ((got.float() - x.float()).abs().amax() < 0.5)
    q = torch.randn(2, 16, dim, device="cuda", dtype=torch.bfloat16)
    got = nv.paged_attention(q, cache, page_table, ints([1050, 1050]), 0.1)
    want, bound = attention(q, cache, page_table, [1050, 1050], 0.1)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_that_nearly_cancel(dtype):
    """Two keys and values of 1 and -1, as codes far from the middle: what is left is the weights' difference, to the terms' precision."""
    cache = nv.PagedCache.new(1, 1, 16, 64, nv.Quant.affine(64, 8), dtype)
    cache.keys.weight.view(torch.int32)[0, 0, 0, 0] = 1
    cache.keys.scales.fill_(1.0)
    cache.values.weight.view(torch.int32).fill_(0x01010101)
    cache.values.scales[0, 0, 0], cache.values.scales[0, 0, 1] = 1.0, -1.0
    q = torch.zeros(32, 1, 64, device="cuda")
    q[:, 0, 0] = torch.rand(32, device="cuda") * 2.0 ** -6
    q = q.to(dtype)
    got = nv.paged_attention(q, cache, torch.zeros(32, 1, dtype=torch.int32, device="cuda"), ints([2] * 32), 1.0)
    # (values are 1 and -1: code 1 is 127 below the middle, so a weight's rounding is seen 127-fold)
    term = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -16}[dtype]
    want = torch.tanh(q[..., :1].double() / 2).expand_as(got)
    assert ((got.double() - want).abs() <= 127 * term + 2.0 ** -8 * want.abs() + 128 * 16 * 2.0 ** -24).all()


def test_captured_attention_follows_its_lengths():
    """One graph over lengths that grow from no split to several, other work between the replays, another graph of the same shapes beside it."""
    page_table, pages = tables([4096, 4096], 64)
    cache = random_cache(pages, 2, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    q = torch.randn(2, 8, 128, device="cuda", dtype=torch.bfloat16)
    lengths = ints([1, 9])
    nv.paged_attention(q, cache, page_table, lengths, 0.1)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(nv.paged_attention(q, cache, page_table, lengths, 0.1))
    for n in (3, 256, 257, 1000, 4096, 2):
        lengths.copy_(ints([n, max(1, n // 2)]))
        q.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = nv.paged_attention(q, cache, page_table, lengths, 0.1)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), n


def test_two_streams_at_once():
    page_table, pages = tables([3000, 2000], 64)
    cache = random_cache(pages, 4, 64, 128, nv.Quant.affine(64, 4), torch.bfloat16)
    qs = [torch.randn(2, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    lengths = ints([3000, 2000])
    want = [nv.paged_attention(q, cache, page_table, lengths, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(nv.paged_attention(qs[i], cache, page_table, lengths, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_a_run_of_them_is_contiguous_attention():
    """Prompt and decode steps through the pages: rope, append and attention together against float64 over what the cache holds, and near
    attention over the exact keys and values."""
    from tests.paged_reference import table
    torch.manual_seed(2)
    heads, key_heads, dim, page = 8, 2, 128, 16
    cache = nv.PagedCache.new(40, key_heads, page, dim, nv.Quant.affine(32, 8))
    rotation = nv.Rotation(table(256, dim))
    page_table = torch.randperm(40, device="cuda").to(torch.int32).reshape(2, 20)
    put = lambda n, h: torch.randn(n, h, dim, device="cuda", dtype=torch.bfloat16)
    lengths = [0, 0]
    held = [[], []]
    for rows in ([37, 70], [1, 1], [1, 1], [5, 1], [1, 30]):
        n = sum(rows)
        q, k, v = put(n, heads), put(n, key_heads), put(n, key_heads)
        sequences = ints([0] * rows[0] + [1] * rows[1])
        positions = ints([*range(lengths[0], lengths[0] + rows[0]), *range(lengths[1], lengths[1] + rows[1])])
        lengths = [a + b for a, b in zip(lengths, rows)]
        turned = nv.append_paged(cache, k, v, page_table, positions, sequences, rotation, q=q)
        assert torch.equal(turned, nv.rope(q.transpose(0, 1)[None], rotation, positions[None])[0].transpose(0, 1))
        starts = [0, rows[0], n]
        got = nv.paged_attention(turned, cache, page_table, ints(lengths), dim ** -0.5, ints(starts), max(rows))
        want, bound = attention(turned, cache, page_table, lengths, dim ** -0.5, starts)
        assert ((got.double() - want).abs() <= bound).all()
        kr = nv.rope(k.transpose(0, 1)[None].float(), rotation, positions[None])[0].transpose(0, 1)
        for b in range(2):
            held[b].append((kr[starts[b]:starts[b + 1]], v[starts[b]:starts[b + 1]].float()))
            kk, vv = (torch.cat([h[i] for h in held[b]]).repeat_interleave(heads // key_heads, 1) for i in range(2))
            s = torch.einsum("nhd,shd->hns", turned[starts[b]:starts[b + 1]].float(), kk) * dim ** -0.5
            hide = torch.arange(lengths[b], device="cuda")[None] > (lengths[b] - rows[b] + torch.arange(rows[b], device="cuda"))[:, None]
            near = torch.einsum("hns,shd->nhd", torch.softmax(s.masked_fill(hide, float("-inf")), -1), vv)
            # eight bits of a range of about 5: half a step is 0.01, of the keys' 128 products 0.01 x |q| / sqrt(128) of a score
            assert (got[starts[b]:starts[b + 1]].float() - near).abs().max() < 0.1
