"""The quantized append to pages and its read (csrc/paged_cache.hip) against 64 bits.

A key is float32 on its way to its code: at most eight roundings (norm and rotation, as tests/test_gpu_heads.py counts them) of the sizes of
its terms, 2^-24 each; call them e.  Of a group: the bias is the end of the range within e and one rounding of the element type, the scale
that of the definition within what e does to a range and a rounding.  A code is the nearest to x of those that the stored scale and bias
allow: |x - (code scale + bias)| <= |scale| / 2 + e (and the float32 difference and quotient's roundings), or x lies outside the codes' range and the code is its end."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY, codes_of, normed, table, turned, wide

pytestmark = pytest.mark.gpu
FORMS = [(128, 64, 4), (128, 32, 4), (128, 128, 8), (64, 64, 4), (64, 32, 8), (128, 64, 8)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def pool(pages, heads, page, dim, group, bits, dtype):
    cache = nv.PagedCache.new(pages, heads, page, dim, nv.Quant.affine(group, bits), dtype)
    for q in (cache.keys, cache.values):  # (what is not written is to stay)
        q.weight.view(torch.int32).fill_(0x5A5A5A5A)
        q.scales.fill_(3.0), q.biases.fill_(-2.0)
    return cache


def rows_of(q, at, heads, page):
    """(page, place) rows as a `Quantized` [tokens, heads, ...]."""
    pick = lambda t: t[at[0], :, at[1]]
    return nv.Quantized(pick(q.weight.view(torch.int32)).contiguous().view(torch.uint32), pick(q.scales), pick(q.biases), q.quant)


def check_codes(stored, x, size, roundings):
    """`stored` rows of float64 values `x`, each off by at most `roundings` 2^-24 of `size`."""
    group, bits, dtype = stored.quant.group_size, stored.quant.bits, stored.scales.dtype
    bins, u = 2 ** bits - 1, HALF[dtype]
    e = roundings * 2.0 ** -24 * size
    c, s, z = codes_of(stored), wide(stored.scales, group), wide(stored.biases, group)
    off = (x - (c * s + z)).abs()
    # (x - bias and its quotient by the scale are float32: 2^-24 each of at most bins + 1 scales)
    within = off <= s.abs() * (0.5 + 2 * 2.0 ** -24 * (bins + 1)) + e
    t = (x - z) / s
    outside = ((c == 0) & (t < 0.5 + 1e-3)) | ((c == bins) & (t > bins - 0.5 - 1e-3))
    assert (within | outside).all(), off.max().item()
    g = lambda v: v.unflatten(-1, (-1, group))
    low, high, slack = g(x).amin(-1), g(x).amax(-1), g(e).amax(-1)
    falls = stored.scales < 0
    edge = torch.where(falls, high, low)
    zero = stored.biases == 0  # (a range that starts at no whole step from 0)
    assert ((stored.biases.double() - edge).abs() <= u * edge.abs() + slack * (1 + u) + TINY[dtype])[~zero].all()
    assert (edge.abs() <= (high - low) / bins / 2 + slack + 2e-7)[zero].all()
    assert ((edge.abs() >= torch.maximum(low.abs(), high.abs()) - slack)).all()
    span = (high - low).clamp_min(1e-7 * bins)
    steps = torch.round(edge.abs() * bins / span)
    want = torch.where(steps == 0, span / bins, edge.abs() / steps.clamp_min(1))
    sure = (edge.abs() * bins / span - steps).abs() < 0.49  # (else either number of steps)
    near = (stored.scales.double().abs() - want).abs() <= (u + 2.0 ** -20) * want + 4 * slack / bins + slack + TINY[dtype]
    assert (near | ~sure).all()


@pytest.mark.parametrize("dim,group,bits", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_append(dim, group, bits, dtype):
    """Ragged sequences over shuffled pages: keys with and without norm and rotation (whole and partial, both layouts), values, queries;
    padding and everything around the rows stays as it was."""
    for page, heads, query_heads, turn, norm, interleaved in ((16, 3, 6, dim, True, False), (64, 1, 4, dim // 2, False, True), (32, 2, 0, 0, True, False), (256, 5, 5, 6, False, False)):
        torch.manual_seed(page + dim)
        each, held = [1, 40, 3, 17], [0, 7, page - 1, 30]
        columns = 5
        cache = pool(4 * columns, heads, page, dim, group, bits, dtype)
        before = [t.clone() for q in (cache.keys, cache.values) for t in (q.weight.view(torch.int32), q.scales, q.biases)]
        page_table = torch.randperm(4 * columns, device="cuda").to(torch.int32).reshape(4, columns)
        positions = torch.cat([torch.arange(h, h + n) for h, n in zip(held, each)]).to(torch.int32).cuda()
        sequences = torch.repeat_interleave(torch.arange(4), torch.tensor(each)).to(torch.int32).cuda()
        positions[[5, 44]] = torch.tensor([-1, -9], dtype=torch.int32, device="cuda")
        tokens = sum(each)
        put = lambda n: (torch.randn(tokens, n, dim, device="cuda") * torch.exp(torch.randn(dim, device="cuda"))).to(dtype)
        k, v, q = put(heads), put(heads), put(query_heads) if query_heads else None
        kw, qw = ((1 + 0.3 * torch.randn(dim, device="cuda")).to(dtype) if norm else None for _ in range(2))
        rotation = nv.Rotation(table(2048, turn), interleaved) if turn else None
        got = nv.append_paged(cache, k, v, page_table, positions, sequences, rotation, kw, q, qw, 1e-6)

        real = positions >= 0
        at_table = positions.clamp_min(0).long()
        def rotated(x, w):
            y = normed(x, w, 1e-6)
            return turned(y, rotation.table[at_table][:, None], interleaved) if rotation else (y, y.abs())
        if q is None:
            assert got is None
        else:
            want, size = rotated(q, qw)
            slack = 8 * 2.0 ** -24 * size
            assert ((got.double() - want).abs() <= HALF[dtype] * (want.abs() + slack) + slack + TINY[dtype]).all()
        at = (page_table[sequences.long(), at_table // page].long()[real], (at_table % page)[real])
        want, size = rotated(k, kw)
        check_codes(rows_of(cache.keys, at, heads, page), want[real], size[real], 8)
        check_codes(rows_of(cache.values, at, heads, page), v.double()[real], torch.zeros_like(v.double()[real]), 0)
        # read back, and nothing else written
        keys, values = nv.read_paged(cache, page_table, positions, sequences)
        for rows, p in ((keys, cache.keys), (values, cache.values)):
            stored = rows_of(p, at, heads, page)
            exact = (codes_of(stored) * wide(stored.scales, group) + wide(stored.biases, group)).float().to(dtype)
            assert torch.equal(rows[real], exact) and (rows[~real] == 0).all()
        for t, b in zip([t for p in (cache.keys, cache.values) for t in (p.weight.view(torch.int32), p.scales, p.biases)], before):
            t[at[0], :, at[1]] = b[at[0], :, at[1]]
            assert torch.equal(t, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_step_is_the_prompt(dtype):
    """A token appended alone has the codes that it has among others, for any strides."""
    torch.manual_seed(3)
    rotation = nv.Rotation(table(128, 128))
    a, b = pool(6, 2, 16, 128, 64, 4, dtype), pool(6, 2, 16, 128, 64, 4, dtype)
    page_table = torch.randperm(6, device="cuda").to(torch.int32).reshape(2, 3)
    wide_rows = torch.randn(40, 5 * 128 + 3, device="cuda").to(dtype)
    k, v = wide_rows[:, :256].unflatten(-1, (2, 128)), wide_rows[:, 258:514].unflatten(-1, (2, 128))
    w = torch.rand(128, device="cuda").to(dtype)
    positions = torch.arange(40, dtype=torch.int32, device="cuda") % 20
    sequences = (torch.arange(40, device="cuda") // 20).to(torch.int32)
    nv.append_paged(a, k, v, page_table, positions, sequences, rotation, w)
    for p in range(20):  # (both sequences' next token)
        at = [p, 20 + p]
        nv.append_paged(b, k[at].contiguous(), v[at].contiguous(), page_table, positions[at], None, rotation, w)
    for x, y in ((a.keys, b.keys), (a.values, b.values)):
        assert torch.equal(x.weight.view(torch.int32), y.weight.view(torch.int32)) and torch.equal(x.scales, y.scales) and torch.equal(x.biases, y.biases)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_of_one_value(bits, dtype):
    """Constants, zeros, tiny and huge ranges, ends of either sign: the ends are exact in the cache's type, the rest within half a step."""
    page_table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cache = pool(1, 1, 16, 64, 32, bits, dtype)
    rows = torch.zeros(8, 1, 64, device="cuda")
    rows[1], rows[2], rows[3] = 5.0, -0.375, 1e-5
    rows[4, 0, ::2], rows[5, 0, 7], rows[6, 0, :32], rows[7] = 1000.0, -3.0, torch.linspace(-4, 4, 32, device="cuda"), torch.randn(64, device="cuda") * 1e-3
    v = rows.to(dtype)
    at = torch.arange(8, dtype=torch.int32, device="cuda")
    nv.append_paged(cache, v, v, page_table, at, torch.zeros_like(at))
    _, got = nv.read_paged(cache, page_table, at, torch.zeros_like(at))
    assert (got[0] == 0).all() and torch.equal(got[1:3], v[1:3]) and torch.equal(got[4].abs().amax(), v[4].abs().amax())
    check_codes(rows_of(cache.values, (torch.zeros(8, dtype=torch.long, device="cuda"), at.long()), 1, 16), v.double(), torch.zeros_like(v.double()), 0)


def test_nan_stays_in_its_group():
    cache = pool(1, 1, 16, 128, 32, 4, torch.bfloat16)
    page_table, at = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    v = torch.randn(1, 1, 128, device="cuda", dtype=torch.bfloat16)
    want = v.clone()
    v[0, 0, 40], v[0, 0, 70] = float("nan"), float("inf")
    nv.append_paged(cache, v, v, page_table, at)
    keys, values = nv.read_paged(cache, page_table, at)
    nv.append_paged(cache, want, want, page_table, at)
    clean, _ = nv.read_paged(cache, page_table, at)
    for got in (keys, values):
        assert torch.equal(got[..., :32], clean[..., :32]) and torch.equal(got[..., 96:], clean[..., 96:])


def test_tokens_outside_the_cache_are_not_written():
    """Positions behind the page table's columns and the angles' table, sequences and pages that are none."""
    cache = pool(4, 1, 16, 64, 64, 4, torch.float16)
    before = cache.keys.weight.view(torch.int32).clone()
    page_table = torch.tensor([[0, 4], [-1, 1]], dtype=torch.int32, device="cuda")
    k = torch.randn(7, 1, 64, device="cuda", dtype=torch.float16)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    positions, sequences = ints(32, 16, 3, 2, 2, 1 << 30, 31), ints(0, 0, 1, 2, -1, 0, 1)
    nv.append_paged(cache, k, k, page_table, positions, sequences, nv.Rotation(table(31, 64)))
    assert torch.equal(cache.keys.weight.view(torch.int32), before) and (cache.values.scales == 3).all()
    keys, values = nv.read_paged(cache, page_table, ints(32, 16, 3, 2, 2, 1 << 30), ints(0, 0, 1, 2, -1, 0))
    assert (keys == 0).all() and (values == 0).all()


def test_nothing_to_do():
    cache = pool(2, 2, 16, 64, 64, 4, torch.bfloat16)
    empty = torch.zeros(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    page_table = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    assert nv.append_paged(cache, empty, empty, page_table, none, none, q=empty).shape == (0, 2, 64)
    assert [t.shape for t in nv.read_paged(cache, page_table, none, none)] == [(0, 2, 64)] * 2
    one = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    nv.append_paged(cache, one, one, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), zero)  # (a table of no columns holds no position)


def test_captured_append_follows_its_positions():
    rotation = nv.Rotation(table(64, 64))
    a, b = pool(8, 2, 16, 64, 32, 4, torch.bfloat16), pool(8, 2, 16, 64, 32, 4, torch.bfloat16)
    page_table = torch.randperm(8, device="cuda").to(torch.int32).reshape(2, 4)
    k, v, q = (torch.randn(2, n, 64, device="cuda", dtype=torch.bfloat16) for n in (2, 2, 4))
    positions = torch.tensor([0, 30], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nv.append_paged(a, k, v, page_table, positions, None, rotation, q=q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nv.append_paged(a, k, v, page_table, positions, None, rotation, q=q)
    for step in range(1, 6):
        for t in (k, v, q):
            t.normal_()
        nv.append_paged(b, k, v, page_table, positions, None, rotation)  # (the first of them is the call on the other stream)
        graph.replay()
        torch.cuda.synchronize()
        want = nv.append_paged(b, k, v, page_table, positions, None, rotation, q=q)
        assert torch.equal(out, want)
        for x, y in ((a.keys, b.keys), (a.values, b.values)):
            assert torch.equal(x.weight.view(torch.int32), y.weight.view(torch.int32)) and torch.equal(x.scales, y.scales)
        positions.add_(5)
