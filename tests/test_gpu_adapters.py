"""Low-rank adapters of many requests (csrc/adapters.hip) against 64 bits."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TERM = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 0.0}  # what two terms of a value leave of it


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(rows, k, n, rank, count, dtype, seed=0, scaled=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    put = lambda *s: torch.randn(s, generator=g, device="cuda")
    adapters = nv.Adapters((put(count, rank, k) * k ** -0.5).to(dtype), put(count, n, rank).to(dtype), (0.5 + put(count).abs()) if scaled else None)
    return put(rows, n).to(dtype), put(rows, k).to(dtype), adapters


def expected(y, x, adapters, ids):
    """(result, bound).  Both products are float32 sums: of L products at most L roundings of 2^-24 of the sum of their sizes.  Between them a value is
    rounded to its terms.  Then the addition, and the rounding of the result."""
    want, slack = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    k, rank = x.shape[-1], adapters.up.shape[2]
    for a in range(adapters.down.shape[0]):
        rows = (ids == a).nonzero()[:, 0]
        if len(rows) == 0:
            continue
        scale = 1.0 if adapters.scales is None else adapters.scales[a].double()
        down, up, xs = adapters.down[a].double().T, adapters.up[a].double().T, x[rows].double()
        t = xs @ down
        off = k * 2.0 ** -24 * (xs.abs() @ down.abs()) + (TERM[y.dtype] + 2.0 ** -23) * t.abs()
        want[rows] += scale * (t @ up)
        slack[rows] += scale * (off @ up.abs() + rank * 2.0 ** -24 * (t.abs() @ up.abs()))
    return want, slack + 2.0 ** -24 * (want.abs() + y.double().abs()) + HALF[y.dtype] * want.abs() + TINY[y.dtype]


def check(y, x, adapters, ids, **more):
    got = nv.apply_adapters(y, x, adapters, ids, **more)
    want, bound = expected(y, x, adapters, ids)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,rank,count", [
    (1, 64, 64, 16, 1), (1, 4096, 1024, 8, 3), (2, 32, 16, 1, 2), (5, 100, 70, 3, 4), (16, 31, 65, 12, 16), (17, 33, 63, 17, 5), (15, 1, 1, 1, 2),
    (64, 512, 300, 32, 64), (100, 257, 129, 64, 7), (33, 96, 64, 100, 3), (7, 64, 40, 256, 2), (40, 2880, 2880, 12, 9), (300, 640, 257, 16, 20)])
def test_sizes(dtype, rows, k, n, rank, count):
    """Odd sizes and tiles' edges, ranks of one to several tiles, each row its own adapter, some none."""
    y, x, adapters = make(rows, k, n, rank, count, dtype)
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-1, count, (rows,), generator=g).to(torch.int32).cuda()
    check(y, x, adapters, ids)
    check(y, x, adapters, torch.full_like(ids, count - 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_of_requests(dtype):
    """Many tiles: prompts of one request each, single tokens between them, enough that a block takes a tile's adapters one after the other."""
    rows = 1500
    y, x, adapters = make(rows, 320, 200, 16, 6, dtype)
    ids = torch.repeat_interleave(ints([0, 3, -1, 5, 1, 1, 4, 0, 2]), ints([700, 1, 90, 1, 1, 400, 300, 5, 2]))
    check(y, x, adapters, ids.contiguous())
    check(y, x, adapters, (torch.arange(rows, device="cuda") % 7 - 1).to(torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_an_adapter_stay(dtype):
    """Ids that are no adapter's, of either sign: the bits of y, whatever x holds there."""
    y, x, adapters = make(40, 128, 96, 16, 3, dtype)
    ids = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    ids[5], ids[7], ids[9], ids[11] = 3, 1 << 30, -(1 << 31), 2
    x[5], x[7], x[0] = float("nan"), float("inf"), float("nan")
    y[3, 4], y[5, 6] = float("inf"), float("nan")
    got = nv.apply_adapters(y, x, adapters, ids)
    stays = torch.ones(40, dtype=torch.bool, device="cuda")
    stays[11] = False
    bits = {2: torch.int16, 4: torch.int32}[y.element_size()]
    assert torch.equal(got[stays].view(bits), y[stays].view(bits))
    want, bound = expected(y[11:12], x[11:12], adapters, ids[11:12])
    assert ((got[11:12].double() - want).abs() <= bound).all()
    none = nv.Adapters(adapters.down[:0], adapters.up[:0], adapters.scales[:0])
    assert torch.equal(nv.apply_adapters(y, x, none, ids).view(bits), y.view(bits))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_and_adapters_keep_to_themselves(dtype):
    """NaN and infinite values of one row's x, and of one adapter's weights, reach that row and that adapter's rows alone."""
    y, x, adapters = make(34, 256, 128, 16, 4, dtype)
    ids = (torch.arange(34, device="cuda") % 4).to(torch.int32)
    x[2], x[17, 5] = float("nan"), float("inf")
    adapters.down[1, 3, 7], adapters.up[1, 5, 2], adapters.up[3, 9, 0] = float("inf"), float("nan"), float("inf")
    got = nv.apply_adapters(y, x, adapters, ids)
    clean = (ids == 0) | (ids == 2)
    clean[2] = False  # (rows 2 and 17: their own x)
    want, bound = expected(y, torch.where(clean[:, None], x, torch.zeros_like(x)), nv.Adapters(*(t[[0, 0, 2, 2]] for t in (adapters.down, adapters.up, adapters.scales))), ids)
    assert ((got.double() - want).abs() <= bound)[clean].all()
    assert not got[2].isfinite().any() and not got[1, 5].isfinite()
    assert not got[3, 9].isfinite() and got[3, 10].isfinite()


@pytest.mark.parametrize("dtype", TYPES)
def test_sizes_of_values(dtype):
    """Values between the products beyond and far below float16's range, results within it."""
    y, x, adapters = make(20, 128, 64, 16, 2, dtype)
    ids = (torch.arange(20, device="cuda") % 2).to(torch.int32)
    adapters.down[0] *= 300
    x[::4] *= 1000  # (products up to some 10^6)
    adapters.up[0] *= 2.0 ** -13
    adapters.scales[0] = 0.01
    adapters.down[1] *= 2.0 ** -12
    adapters.scales[1] = 2.0 ** 10
    check(y, x, adapters, ids)


def test_strides_places_and_shapes():
    """Views with strides between the rows, leading dimensions, the result in place of y, in a view, and into another tensor."""
    for dtype in TYPES:
        y, x, adapters = make(24, 96, 80, 8, 3, dtype)
        ids = (torch.arange(24, device="cuda") % 4 - 1).to(torch.int32)
        want = check(y, x, adapters, ids)
        wide = torch.randn(24, 300, device="cuda").to(dtype)
        wide[:, 7:103], wide[:, 110:190] = x, y
        assert torch.equal(nv.apply_adapters(wide[:, 110:190], wide[:, 7:103], adapters, ids), want)
        turned = x.T.contiguous().T
        assert torch.equal(nv.apply_adapters(y, turned, adapters, ids), want)
        assert torch.equal(nv.apply_adapters(y.view(2, 3, 4, 80), x.view(2, 3, 4, 96), adapters, ids.view(2, 3, 4)), want.view(2, 3, 4, 80))
        before = wide.clone()
        assert nv.apply_adapters(wide[:, 110:190], x, adapters, ids, out=wide[:, 110:190]).data_ptr() == wide[:, 110:190].data_ptr()
        assert torch.equal(wide[:, 110:190], want) and torch.equal(wide[:, :110], before[:, :110]) and torch.equal(wide[:, 190:], before[:, 190:])
        same = y.clone()
        assert nv.apply_adapters(same, x, adapters, ids, out=same) is same and torch.equal(same, want)
        one = x[:1].expand(24, 96)
        assert torch.equal(nv.apply_adapters(y, one, adapters, ids), nv.apply_adapters(y, one.contiguous(), adapters, ids))
        assert nv.apply_adapters(y[0], x[0], adapters, ids[1:2].reshape(())).shape == (80,)
        assert torch.equal(nv.apply_adapters(y, x, nv.Adapters(adapters.down, adapters.up, None), ids),
                           nv.apply_adapters(y, x, nv.Adapters(adapters.down, adapters.up, torch.ones(3, device="cuda")), ids))


def test_calls_of_nothing():
    y, x, adapters = make(4, 64, 32, 8, 2, torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert nv.apply_adapters(y[:0], x[:0], adapters, none).shape == (0, 32)


def test_captured_calls_follow_their_ids():
    """Two graphs of one call, whose ids and rows change between the replays, beside eager work on the same operands."""
    y, x, adapters = make(70, 512, 256, 16, 8, torch.bfloat16)
    ids = torch.zeros(70, dtype=torch.int32, device="cuda")
    outs = [torch.zeros_like(y) for _ in range(2)]
    nv.apply_adapters(y, x, adapters, ids)
    graphs = [torch.cuda.CUDAGraph() for _ in outs]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            nv.apply_adapters(y, x, adapters, ids, out=out)
    for step in range(5):
        ids.copy_(torch.randint(-1, 8, (70,)).to(torch.int32).sort().values if step % 2 else torch.randint(-1, 8, (70,)).to(torch.int32))
        x.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = check(y, x, adapters, ids)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_two_streams_at_once():
    sets = [make(50, 1024, 512, 16, 8, torch.bfloat16, seed=i) for i in range(2)]
    ids = (torch.arange(50, device="cuda") % 9 - 1).to(torch.int32)
    want = [nv.apply_adapters(*s, ids) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(nv.apply_adapters(*sets[i], ids))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
