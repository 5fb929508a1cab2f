"""Rotary positions with several axes (time, height, width): `rope`, `head_norm_rope`, `append_paged`."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY, normed, table, turned

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def angles(rotation, positions):
    """[batch, length, pairs, 2] of int32 positions [axes, batch, length], clamped to the table."""
    rows = rotation.table.shape[0]
    pair = torch.arange(len(rotation.axes), device="cuda")
    return rotation.table[positions.long().clamp(0, rows - 1)[list(rotation.axes)].permute(1, 2, 0), pair]


def check(got, x, weight, rotation, positions, eps=1e-6):
    """Two float32 products and a sum of them for each value, three roundings with a norm; then the result's own."""
    y, size = turned(normed(x, weight, eps), angles(rotation, positions)[:, None], rotation.interleaved)
    bound = 5 * 2.0 ** -24 * size + HALF[x.dtype] * y.abs() + TINY[x.dtype]
    assert ((got.double() - y).abs() <= bound).all()


def make(sections, dealt, interleaved, positions=300):
    axes = nv.rotary_axes(sections, dealt)
    return nv.Rotation(table(positions, 2 * len(axes)), interleaved, axes)


def places(count, b, l, high=300, seed=0):
    return torch.randint(0, high, (count, b, l), generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,sections,dealt", [
    (128, (24, 20, 20), True), (128, (16, 24, 24), False), (64, (0, 16, 16), False), (80, (20, 20), False), (80, (3, 7, 9), True), (50, (1, 2, 3, 4), False),
    (7, (1, 2), True), (128, (64,), False), (512, (100, 56, 50, 50), True), (200, (1, 1, 60), True), (96, (5, 0, 11), False)])
def test_rope(dtype, interleaved, dim, sections, dealt):
    """Pairs in consecutive runs and dealt out, runs that cross a lane's eight values, parts of heads, one to four axes."""
    rotation = make(sections, dealt, interleaved)
    for b, h, l in ((1, 1, 1), (2, 3, 5), (3, 2, 70)):
        x = torch.randn(b, l, h, dim, device="cuda").to(dtype).transpose(1, 2)
        at = places(len(sections), b, l)
        check(nv.rope(x, rotation, at), x, None, rotation, at)
        same = x.clone()
        assert nv.rope(same, rotation, at, out=same) is same
        assert torch.equal(same, nv.rope(x, rotation, at))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_norms(dtype, interleaved):
    for dim, sections in ((128, (24, 20, 20)), (80, (8, 8, 8)), (64, (11, 11, 10))):
        rotation = make(sections, True, interleaved)
        q, k = (torch.randn(2, 33, h, dim, device="cuda").to(dtype).transpose(1, 2) for h in (5, 2))
        w = (1 + 0.2 * torch.randn(dim, device="cuda")).to(dtype)
        at = places(3, 2, 33)
        for weights in ((w, None), (None, w), (w, w.flip(0))):
            got = nv.head_norm_rope(q, k, *weights, rotation, at)
            for y, x, weight in zip(got, (q, k), weights):
                check(y, x, weight, rotation, at)


@pytest.mark.parametrize("dtype", TYPES)
def test_axes_that_move_together_are_one_position(dtype):
    """Bit for bit the plain rotation; ints and offsets of a rotation with axes are every axis's position."""
    rotation = make((24, 20, 20), True, False)
    plain = nv.Rotation(rotation.table)
    x = torch.randn(2, 4, 40, 128, device="cuda").to(dtype)
    at = places(1, 2, 40)[0]
    want = nv.rope(x, plain, at)
    assert torch.equal(nv.rope(x, rotation, at.expand(3, 2, 40).contiguous()), want)
    assert torch.equal(nv.rope(x, rotation, at.expand(4, 2, 40)), want)  # (a fourth axis without pairs, a view)
    assert torch.equal(nv.rope(x, rotation, at), want)
    assert torch.equal(nv.rope(x, rotation, 7), nv.rope(x, plain, 7))
    assert torch.equal(nv.rope(x, rotation, ints([3, 9])), nv.rope(x, plain, ints([3, 9])))


def test_positions_outside_the_table_are_clamped():
    rotation = make((10, 11, 11), False, False)
    x = torch.randn(1, 2, 6, 64, device="cuda")
    at = ints([[[-1, 0, 300, 1 << 30, 5, -(1 << 31)]], [[1, 2, 3, 4, 1000, 6]], [[299, 300, 301, -7, 0, 1]]])
    check(nv.rope(x, rotation, at), x, None, rotation, at)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits,dim,interleaved", [(4, 128, False), (8, 64, True), (4, 64, False)])
def test_append(dtype, bits, dim, interleaved):
    """The keys that the cache holds are those of keys turned beforehand (in float32), and the queries those of `rope`; places and angles differ."""
    torch.manual_seed(1)
    pairs = dim // 2
    rotation = make((pairs - 2 * (pairs // 3), pairs // 3, pairs // 3), True, interleaved)
    tokens, heads, key_heads, page = 45, 6, 2, 16
    caches = [nv.PagedCache.new(8, key_heads, page, dim, nv.Quant.affine(32, bits), dtype) for _ in range(2)]
    page_table = torch.randperm(8, device="cuda").to(torch.int32).reshape(2, 4)
    sequences = (torch.arange(tokens, device="cuda") % 2).to(torch.int32)
    positions = (torch.arange(tokens, device="cuda") // 2).to(torch.int32)
    positions[5] = -1
    q, k, v = (torch.randn(tokens, h, dim, device="cuda").to(dtype) for h in (heads, key_heads, key_heads))
    w = (1 + 0.2 * torch.randn(dim, device="cuda")).to(dtype)
    at = places(3, 1, tokens)[:, 0]
    at[1, 9], at[2, 11] = 300, -1  # (outside the table: not written)
    got = nv.append_paged(caches[0], k, v, page_table, positions, sequences, rotation, w, q, w, rotary_positions=at)
    turn = lambda x: nv.head_norm_rope(x.transpose(0, 1)[None], x.transpose(0, 1)[None], w, w, rotation, at[:, None].contiguous())[0][0].transpose(0, 1)
    assert torch.equal(got, turn(q))
    keys, values = nv.read_paged(caches[0], page_table, positions, sequences)
    lost = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    lost[[5, 9, 11]] = True
    assert (keys[lost] == 0).all() and (values[lost] == 0).all()
    y, _ = turned(normed(k, w, 1e-6), angles(rotation, at[:, None])[0][:, None], interleaved)
    # The bias is the end e of a group's range that is further from 0, the step |e| / s with s the whole number nearest to |e| (2^bits - 1) / span, which is
    # (2^bits - 1) / 2 at least.  A code is the nearest of 2^bits; where s was rounded up by as much as a half the codes' reach, (2^bits - 1) steps, is short of the
    # other end by span x 0.5 / (s + 0.5) < span / (2^bits - 1), which is more than half a step.  Scale and bias are rounded to the type.
    grouped = y.unflatten(-1, (-1, 32))
    span = (grouped.amax(-1) - grouped.amin(-1)).repeat_interleave(32, -1)
    most = grouped.abs().amax(-1).repeat_interleave(32, -1)
    bound = span / (2 ** bits - 1) + 2 * HALF[dtype] * (most + span) + HALF[dtype] * y.abs() + 1e-6
    assert ((keys.double() - y).abs() <= bound)[~lost].all()
    # values as without any rotation
    kept = torch.where(lost, -1, positions)
    nv.append_paged(caches[1], k, v, page_table, kept, sequences)
    assert torch.equal(values, nv.read_paged(caches[1], page_table, kept, sequences)[1])


def test_append_with_one_axis_of_positions_of_their_own():
    """Positions shifted against the places: those of the plain call whose places are so."""
    torch.manual_seed(2)
    rotation = nv.Rotation(table(300, 64))
    caches = [nv.PagedCache.new(4, 2, 16, 64, nv.Quant.affine(64, 8)) for _ in range(2)]
    page_table, shifted = ints([[2, 0, 1, 3]]), ints([[9, 2, 0, 1, 3]])
    k, v, q = (torch.randn(30, 2, 64, device="cuda").bfloat16() for _ in range(3))
    positions, sequences = torch.arange(30, dtype=torch.int32, device="cuda"), torch.zeros(30, dtype=torch.int32, device="cuda")
    one = nv.append_paged(caches[0], k, v, page_table, positions, sequences, rotation, q=q, rotary_positions=positions + 16)
    other = nv.append_paged(caches[1], k, v, shifted, positions + 16, sequences, rotation, q=q)
    assert torch.equal(one, other)
    for a, b in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
        assert torch.equal(a.weight.view(torch.int32), b.weight.view(torch.int32)) and torch.equal(a.scales, b.scales) and torch.equal(a.biases, b.biases)


def test_captured_calls_follow_their_positions():
    rotation = make((24, 20, 20), True, False)
    x, at = torch.randn(2, 8, 30, 128, device="cuda").bfloat16(), places(3, 2, 30)
    out = torch.zeros_like(x)
    nv.rope(x, rotation, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nv.rope(x, rotation, at, out=out)
    for i in range(4):
        at.copy_(places(3, 2, 30, seed=i + 1))
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nv.rope(x, rotation, at))
        check(out, x, None, rotation, at)
