"""Rotary positions and norms of heads (csrc/heads.hip) against 64 bits.  Bounds, u half a step of the element type: the rotation makes
three float32 roundings of terms as large as |x c| + |p n| (2^-23 of their sum), the norm three more before it (the factor's, its product's, the
weight's), then one rounding of the result."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY, normed, table, turned

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, size, roundings):
    u = HALF[got.dtype]
    slack = roundings * 2.0 ** -24 * size
    assert ((got.double() - want).abs() <= u * (want.abs() + slack) + slack + TINY[got.dtype]).all(), (got.double() - want).abs().max().item()


def angles(rotation, b, l, offset):
    if isinstance(offset, int):
        at = offset + torch.arange(l, device="cuda").expand(b, l)
    else:
        at = offset.long()[:, None] + torch.arange(l, device="cuda") if offset.ndim == 1 else offset.long()
    return rotation.table[at.clamp(0, rotation.table.shape[0] - 1)][:, None]


@pytest.mark.parametrize("dim,dims", [(128, 128), (64, 64), (128, 64), (80, 32), (96, 38), (256, 256), (7, 6), (1, 0), (512, 16), (200, 130), (130, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rope(dim, dims, interleaved, dtype):
    """Whole and partial heads, sizes that are runs of eight and that are not, one token and ragged numbers, all three kinds of offsets."""
    torch.manual_seed(dim + dims)
    rotation = nv.Rotation(table(700, dims), interleaved) if dims else nv.Rotation(torch.zeros(700, 0, 2, device="cuda"))
    for b, h, l in ((1, 1, 1), (3, 5, 17), (2, 33, 100)):
        x = torch.randn(b, h, l, dim, device="cuda").to(dtype)
        per = torch.randint(0, 600, (b,), device="cuda", dtype=torch.int32)
        each = torch.randint(0, 700, (b, l), device="cuda", dtype=torch.int32)
        for offset in (5, per, each):
            want, size = turned(x.double(), angles(rotation, b, l, offset), interleaved)
            close(nv.rope(x, rotation, offset), want, size, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,dims", [(128, 2), (128, 14), (128, 16), (128, 18), (128, 50), (128, 126), (64, 24), (64, 62), (80, 40), (256, 102), (512, 510), (8, 6)])
def test_partners_across_runs(dim, dims, dtype):
    """Heads of whole runs of eight whose halves are not: every place of a half's end in a run; what stays is infinite and NaN; the norm before it."""
    torch.manual_seed(dim + dims)
    for interleaved in (False, True):
        rotation = nv.Rotation(table(300, dims), interleaved)
        x = torch.randn(2, 61, 5, dim, device="cuda").to(dtype).transpose(1, 2)
        want, size = turned(x.double(), angles(rotation, 2, 61, 3), interleaved)
        close(nv.rope(x, rotation, 3), want, size, 3)
        w = (1 + 0.3 * torch.randn(dim, device="cuda")).to(dtype)
        for got, weight in zip(nv.head_norm_rope(x, x, w, None, rotation, 3), (w, None)):
            want, size = turned(normed(x, weight, 1e-6), angles(rotation, 2, 61, 3), interleaved)
            close(got, want, size, 8)
        x = x.clone()
        x[..., dims:] = torch.tensor([float("inf"), float("nan")], device="cuda").repeat(256)[:dim - dims].to(dtype)
        y = nv.rope(x, rotation, 3)
        bits = torch.int32 if dtype == torch.float32 else torch.int16
        assert torch.equal(y[..., dims:].contiguous().view(bits), x[..., dims:].contiguous().view(bits)) and y[..., :dims].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 80, 50])
def test_rope_layouts(dtype, dim):
    """Tokens outermost, a slice of a wider projection, rows at odd addresses, every second head; the results' own strides; in place."""
    torch.manual_seed(dim)
    rotation = nv.Rotation(table(300, 2 * (dim // 4)))
    wide = torch.randn(2, 40, 3 * 6 * dim + 1, device="cuda").to(dtype)
    views = [torch.randn(2, 40, 6, dim, device="cuda").to(dtype).transpose(1, 2), wide[..., :6 * dim].unflatten(-1, (6, dim)).transpose(1, 2),
             wide[..., 1:6 * dim + 1].unflatten(-1, (6, dim)).transpose(1, 2), wide[..., :6 * dim].unflatten(-1, (6, dim))[:, :, ::2].transpose(1, 2),
             wide[:1, :, :6 * dim].unflatten(-1, (6, dim)).transpose(1, 2).expand(3, 6, 40, dim)]
    for x in views:
        want, size = turned(x.double(), angles(rotation, x.shape[0], 40, 9), False)
        got = nv.rope(x, rotation, 9)
        close(got, want, size, 3)
        out = torch.full((x.shape[0], 40, x.shape[1], dim + 8), 7.0, device="cuda", dtype=dtype)
        to = out[..., :dim].transpose(1, 2)
        assert nv.rope(x, rotation, 9, out=to) is to
        assert torch.equal(to, got) and (out[..., dim:] == 7).all()
    x = views[0].clone()
    got = nv.rope(x, rotation, 9)
    nv.rope(x, rotation, 9, out=x)
    assert torch.equal(x, got)


def test_values_that_stay():
    """Behind the rotary values heads are copied bit for bit, infinities and NaN in them too, and do not reach those that turn."""
    rotation = nv.Rotation(table(8, 32))
    for dim in (64, 50):
        x = torch.randn(1, 2, 8, dim, device="cuda", dtype=torch.bfloat16)
        x[..., 32:40] = float("inf")
        x[..., 40:48] = float("nan")
        y = nv.rope(x, rotation)
        assert torch.equal(y[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16)) and y[..., :32].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,dims", [(128, 128), (64, 32), (256, 256), (96, 50), (33, 0), (320, 64)])
def test_head_norm_rope(dtype, dim, dims):
    torch.manual_seed(dim)
    rotation = nv.Rotation(table(500, dims), dims == 32) if dims else None
    for b, h, hk, l in ((1, 1, 1, 1), (3, 8, 2, 19), (16, 32, 8, 1), (2, 5, 7, 90)):
        q, k = (torch.randn(b, l, n, dim, device="cuda").to(dtype).transpose(1, 2) * 3 for n in (h, hk))
        wq, wk = ((1 + torch.randn(dim, device="cuda")).to(dtype) for _ in range(2))
        offset = torch.randint(0, 400, (b,), device="cuda", dtype=torch.int32)
        for a, c in ((wq, wk), (None, wk), (wq, None)):
            for got, x, w in zip(nv.head_norm_rope(q, k, a, c, rotation, offset, 1e-5), (q, k), (a, c)):
                want = normed(x, w, 1e-5)
                want, size = turned(want, angles(rotation, b, l, offset), rotation.interleaved) if rotation else (want, want.abs())
                close(got, want, size, 8)


def test_norm_of_zeros_and_large_values():
    """Zeros stay zeros; squares that float32 does not hold are summed all the same."""
    x = torch.zeros(1, 1, 2, 128, device="cuda")
    x[0, 0, 1] = 2e30
    w = torch.ones(128, device="cuda")
    y, _ = nv.head_norm_rope(x, x, w, w)
    assert (y[0, 0, 0] == 0).all() and (y[0, 0, 1] - 1).abs().max() < 1e-6


def test_positions_outside_the_table_are_clamped():
    rotation = nv.Rotation(table(10, 64))
    x = torch.randn(1, 3, 3, 64, device="cuda")
    at = lambda *p: torch.tensor([p], dtype=torch.int32, device="cuda")
    assert torch.equal(nv.rope(x, rotation, at(-7, 1 << 30, 5)), nv.rope(x, rotation, at(0, 9, 5)))


@pytest.mark.parametrize("dims,base,magnitude", [(128, 10000.0, 1.0), (64, 500000.0, 1.25), (6, 100.0, 1.0)])
def test_rotation_table(dims, base, magnitude):
    """Every angle within 2^-24 of its cosine and sine (64-bit angles: their own error at position 131071 is 2^-36), given frequencies likewise."""
    t = nv.Rotation.new(dims, 131072, base=base, magnitude=magnitude).table
    assert (t.double() - table(131072, dims, magnitude, base).double()).abs().max() <= 2.0 ** -23 * magnitude
    freqs = base ** (torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims) * 3
    angle = torch.arange(5000, dtype=torch.float64, device="cuda")[:, None] * 0.5 / freqs.float().double()
    t = nv.Rotation.new(dims, 5000, scale=0.5, freqs=freqs.float()).table
    assert (t.double() - torch.stack([angle.cos(), angle.sin()], -1)).abs().max() <= 2.0 ** -24


def test_many_heads_and_tokens():
    """More heads than a block takes and more blocks than the chip holds: every one of 2^15 x 40 heads."""
    rotation = nv.Rotation(table(32768, 64))
    x = torch.randn(1, 40, 32768, 64, device="cuda", dtype=torch.bfloat16)
    want, size = turned(x.double(), rotation.table[None, None], False)
    close(nv.rope(x, rotation), want, size, 3)


def test_streams_and_graphs():
    rotation = nv.Rotation(table(64, 128))
    x = torch.randn(4, 8, 1, 128, device="cuda", dtype=torch.bfloat16)
    offset = torch.arange(4, dtype=torch.int32, device="cuda")
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = nv.rope(x, rotation, offset)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, nv.rope(x, rotation, offset))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = nv.head_norm_rope(x, x, w, w, rotation, offset)
    for step in range(4):
        offset.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((y, z), nv.head_norm_rope(x, x, w, w, rotation, offset)):
            assert torch.equal(got, want), step
