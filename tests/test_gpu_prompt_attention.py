"""Attention of whole prompts over dense keys and values (csrc/prompt_kernel.h) against 64 bits."""
import ctypes as C

import pytest
import torch

import nuvec_amd as nv
from nuvec_amd import _lib
from tests.paged_reference import HALF, TINY

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALVES = TYPES[:2]
# What the terms of a weight leave of it (half a step of 11 bits, of 22), and of a weight or, bfloat16's held as float16, a value below float16's normal range.
TERM = {torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -22, torch.float32: 0.0}
SMALL = {torch.bfloat16: 2.0 ** -25, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def expected(q, k, v, scale, rows, lengths, sinks=None, causal=True, window=0):
    """(result, bound) of the sequences' rows in 64 bits.

    Scores are float32 sums of dim products, at most dim roundings of 2^-24 of the sum of their sizes; an error e of them moves the result by at most
    2 e max |v|.  A weight has a few roundings of its own and of its exponent (2^-24 of the score's size), and its terms'; the weighted sums one for each
    product of 16 keys, the weights' sum one for every second key.  A weight, beside a largest one of at least 1, and a value, beside a largest one of at least
    2^-3 (paragraph on bfloat16 in the kernel), that is below float16's normal range is off by half of its smallest step.  Then the result's own rounding."""
    dtype, heads, dim = q.dtype, q.shape[1], q.shape[2]
    rep = heads // k.shape[1]
    want, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    at = key_at = 0
    for n, length in zip(rows, lengths):
        if n > 0 and length > 0:
            x = q[at:at + n].double().transpose(0, 1)
            ks, vs = (t[key_at:key_at + length].double().transpose(0, 1).repeat_interleave(rep, 0) for t in (k, v))
            last = (length - n + torch.arange(n, device=q.device))[:, None] if causal else torch.full((n, 1), length - 1, device=q.device)
            key = torch.arange(length, device=q.device)
            hidden = key > last
            if window:
                hidden = hidden | (key <= last - window)
            scores = (scale * x @ ks.transpose(1, 2)).masked_fill(hidden, float("-inf"))
            sizes = (abs(scale) * x.abs() @ ks.abs().transpose(1, 2)).masked_fill(hidden, 0.0)
            if sinks is not None:
                scores = torch.cat([scores, sinks.double()[:, None, None].expand(heads, n, 1)], -1)
            p = torch.softmax(scores, -1)[..., :length].nan_to_num(0.0)
            y, size, most = p @ vs, p @ vs.abs(), vs.abs().amax((1, 2))[:, None, None]
            e = dim * 2.0 ** -24 * sizes.amax(-1, keepdim=True)
            off = 2 * e * most + (TERM[dtype] + (length / 16 + 64 + 4 * sizes.amax(-1, keepdim=True)) * 2.0 ** -24) * size
            off = off + SMALL[dtype] * (vs.abs().sum(1, keepdim=True) + (8 * most if dtype == torch.bfloat16 else 0.0))
            off = off + ((length / 2 + 64) * 2.0 ** -24 + HALF[dtype]) * y.abs() + TINY[dtype]
            want[at:at + n], bound[at:at + n] = y.transpose(0, 1), off.transpose(0, 1)
        at, key_at = at + n, key_at + length
    return want, bound


def make(rows, keys, heads, key_heads, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    put = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    return put(rows, heads, dim), put(keys, key_heads, dim), put(keys, key_heads, dim)


def check(dtype, heads, key_heads, dim, rows, lengths=None, sinks=False, scale=None, **more):
    lengths = rows if lengths is None else lengths
    q, k, v = make(sum(rows), sum(lengths), heads, key_heads, dim, dtype, seed=sum(lengths) + dim)
    sinks = torch.randn(heads, device="cuda").to(dtype) if sinks else None
    scale = dim ** -0.5 if scale is None else scale
    got = nv.prompt_attention(q, k, v, scale, ints(starts_of(rows)), ints(starts_of(lengths)), sinks, **more)
    want, bound = expected(q, k, v, scale, rows, lengths, sinks, **more)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (dtype, rows, lengths, (off - bound).max().item(), (off / bound).max().item())
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 24, 64, 72, 80, 96, 104, 128, 136, 192, 256])
def test_head_sizes(dtype, dim):
    check(dtype, 4, 2, dim, [37])
    check(dtype, 3, 1, dim, [70, 1, 130], [70, 90, 200], sinks=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rep,rows", [(1, 1), (1, 31), (1, 32), (1, 33), (4, 1), (4, 31), (4, 32), (4, 33), (1, 127), (1, 128), (1, 129), (3, 43), (7, 19), (8, 17), (5, 77), (64, 3)])
def test_lines_at_the_edges_of_blocks(dtype, rep, rows):
    for length in (rows, rows + 45, max(rows - 1, 1), 1):
        check(dtype, rep, 1, 64, [rows], [length])
    check(dtype, 2 * rep, 2, 128, [rows, 1, 0, 2, rows], [rows + 100, 64, 70, 0, rows], sinks=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 300])
def test_lengths_at_the_edges_of_tiles(dtype, length):
    check(dtype, 4, 1, 64, [5], [length])
    check(dtype, 2, 1, 96, [length])
    check(dtype, 2, 2, 128, [3], [length], causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_rows_over_many_keys(dtype, dim):
    """Keys are split over blocks and their states merged; single tokens; splits that see nothing."""
    check(dtype, 4, 2, dim, [1], [3000])
    check(dtype, 4, 1, dim, [1, 7, 40], [5000, 2049, 300], sinks=True)
    check(dtype, 2, 1, dim, [300], [1500])
    check(dtype, 4, 2, dim, [50], [4000], window=70)
    check(dtype, 4, 2, dim, [50], [2000], causal=False)
    check(dtype, 1, 1, dim, [600, 80], [500, 3])  # (rows that see nothing)


@pytest.mark.parametrize("dtype", HALVES)
def test_long_prompts(dtype):
    check(dtype, 8, 2, 128, [1500])
    check(dtype, 8, 2, 64, [900, 1200, 33], [900, 2000, 700])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 200, 1 << 40])
def test_windows(dtype, window):
    check(dtype, 4, 2, 64, [300, 20], [300, 400], window=window)
    check(dtype, 2, 1, 128, [150], [150], window=window, sinks=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales(dtype):
    """Large ones (weights of one key), small ones, none, negative ones."""
    for scale in (3.0, 1e-3, 0.0, -0.2):
        check(dtype, 4, 2, 64, [90], [200], scale=scale)


def test_more_sequences_than_a_wavefront_has_lanes():
    g = torch.Generator().manual_seed(4)
    rows = torch.randint(0, 4, (150,), generator=g).tolist()
    lengths = [n + int(torch.randint(0, 90, (1,), generator=g)) for n in rows]
    rows[5], lengths[5], rows[70], lengths[70], rows[149], lengths[149] = 200, 900, 133, 133, 65, 2000
    check(torch.bfloat16, 8, 2, 128, rows, lengths)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_sequence_without_starts(dtype):
    q, k, v = make(60, 200, 4, 2, 64, dtype)
    want, bound = expected(q, k, v, 0.125, [60], [200])
    one = nv.prompt_attention(q, k, v, 0.125)
    assert ((one.double() - want).abs() <= bound).all()
    assert torch.equal(one, nv.prompt_attention(q, k, v, 0.125, ints([0, 60]), ints([0, 200])))
    k, v = k[:60], v[:60]
    assert torch.equal(nv.prompt_attention(q, k, v, 0.125, ints([0, 20, 60])), nv.prompt_attention(q, k, v, 0.125, ints([0, 20, 60]), ints([0, 20, 60])))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Heads of one fused projection, heads outermost, values at odd addresses, an output between other rows."""
    rows, heads, key_heads, dim = 150, 6, 2, 72
    q, k, v = make(rows, rows, heads, key_heads, dim, dtype)
    want = nv.prompt_attention(q, k, v, 0.1)
    fused = torch.zeros(rows, heads + 2 * key_heads, dim, device="cuda", dtype=dtype)
    fused[:, :heads], fused[:, heads:-key_heads], fused[:, -key_heads:] = q, k, v
    assert torch.equal(nv.prompt_attention(fused[:, :heads], fused[:, heads:-key_heads], fused[:, -key_heads:], 0.1), want)
    outer = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(nv.prompt_attention(*outer, 0.1), want)
    odd = [torch.zeros(t.numel() + 1, device="cuda", dtype=dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(nv.prompt_attention(*odd, 0.1), want)
    last = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(nv.prompt_attention(*last, 0.1), want)
    same = [t[:1].expand_as(t) for t in (k, v)]
    assert torch.equal(nv.prompt_attention(q, *same, 0.1), nv.prompt_attention(q, *(t.contiguous() for t in same), 0.1))
    wide = torch.full((rows, heads, dim + 10), 7.0, device="cuda", dtype=dtype)
    assert nv.prompt_attention(q, k, v, 0.1, out=wide[..., 3:dim + 3]).data_ptr() == wide[..., 3:].data_ptr()
    assert torch.equal(wide[..., 3:dim + 3], want) and (wide[..., :3] == 7).all() and (wide[..., dim + 3:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_the_sequences_stay(dtype):
    q, k, v = make(100, 100, 4, 2, 64, dtype)
    out = torch.full_like(q, 7.0)
    nv.prompt_attention(q, k, v, 0.1, ints([10, 30, 60]), ints([5, 25, 80]), out=out)
    assert (out[:10] == 7).all() and (out[60:] == 7).all()
    want, bound = expected(q[10:60], k[5:80], v[5:80], 0.1, [20, 30], [20, 55])
    assert ((out[10:60].double() - want).abs() <= bound).all()
    nv.prompt_attention(q, k, v, 0.1, ints([0, 0, 0]), ints([0, 0, 0]), out=out.fill_(7.0))
    assert (out == 7).all()
    nv.prompt_attention(q, k[:0], v[:0], 0.1, out=out)
    assert (out == 0).all()
    assert nv.prompt_attention(q[:0], k, v, 0.1).shape == (0, 4, 64)
    # starts outside the operands are clamped to them
    nv.prompt_attention(q, k, v, 0.1, ints([-5, 40, 1 << 30]), ints([-3, 40, 1 << 30]), out=out.fill_(7.0))
    want, bound = expected(q, k, v, 0.1, [40, 60], [40, 60])
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,length", [(64, 100), (128, 200), (256, 70)])
def test_what_is_not_seen_may_hold_anything(dtype, dim, length):
    """NaN and infinite keys and values behind a row, outside its window, and of the neighbouring sequences."""
    q, k, v = make(length, length, 4, 2, dim, dtype)
    want, bound = expected(q, k, v, 0.1, [length], [length], window=40)
    bad = length - 30  # (the key that the last 30 rows see, and the others do not)
    for kind in (float("nan"), float("inf"), -float("inf")):
        for t in (k, v):
            kept = t[bad].clone()
            t[bad] = kind
            got = nv.prompt_attention(q, k, v, 0.1, window=40)
            t[bad] = kept
            assert ((got.double() - want).abs() <= bound)[:bad].all(), kind
    kept = k.clone(), v.clone()
    for at in range(0, length, 3):  # sequences of three keys, of which the middle one is anything
        pass
    rows = [20, 30, length - 50]
    want, bound = expected(q, k, v, 0.1, rows, rows)
    k[20:50], v[20:50] = float("nan"), float("inf")
    got = nv.prompt_attention(q, k, v, 0.1, ints(starts_of(rows)))
    good = torch.ones(length, dtype=torch.bool, device="cuda")
    good[20:50] = False
    assert ((got.double() - want).abs() <= bound)[good].all() and got[20:50].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_values_reach_the_rows_that_see_them(dtype):
    """A value of a kind in one place: that place of the rows behind it, and nothing else."""
    for dim in (64, 128):
        q, k, v = make(150, 150, 4, 2, dim, dtype)
        want, bound = expected(q, k, v, 0.1, [150], [150])
        v[20, 0, 5], v[70, 0, 6], v[90, 1, 7], v[100, 1, 40], v[130, 1, 40] = float("inf"), -float("inf"), float("nan"), float("inf"), -float("inf")
        got = nv.prompt_attention(q, k, v, 0.1)
        clean = torch.ones(got.shape, dtype=torch.bool, device="cuda")
        clean[20:, :2, 5], clean[70:, :2, 6], clean[90:, 2:, 7], clean[100:, 2:, 40] = False, False, False, False
        assert ((got.double() - want).abs() <= bound)[clean].all()
        inf = float("inf")
        assert (got[20:, :2, 5] == inf).all() and (got[70:, :2, 6] == -inf).all() and got[90:, 2:, 7].isnan().all()
        assert (got[100:130, 2:, 40] == inf).all() and got[130:, 2:, 40].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_in_the_scores(dtype):
    """Keys whose scores are minus infinity, or all far below: weights of the others; infinite queries give NaN in their own rows alone."""
    q, k, v = make(40, 80, 2, 1, 64, dtype)
    q, k = q.abs() + 1, k.abs()
    q[7, 1] = float("inf")
    k[10:20, 0, 0] = -float("inf")
    got = nv.prompt_attention(q, k, v, 0.1)
    keep = [i for i in range(80) if not 10 <= i < 20]
    want, bound = expected(q, k[keep], v[keep], 0.1, [40], [70])
    good = torch.ones(40, 2, dtype=torch.bool, device="cuda")
    good[7, 1] = False
    assert ((got.double() - want).abs() <= bound)[good].all() and got[7, 1].isnan().all()
    far = -k * (60.0 if dtype == torch.float16 else 2.0 ** 60)
    far[10:20] = far[0]
    q = q.nan_to_num(posinf=2.0)
    got = nv.prompt_attention(q, far[:, :, :], v, 1.0)
    assert got.isfinite().all() and (got.abs().sum((1, 2)) > 0).all()


def test_sizes_of_values():
    """bfloat16 values far from 1, first tiles of zeros, of small and of large ones in front of others: results as near as their own rounding."""
    for first, rest in ((1e-30, 1e-30), (1e30, 1e30), (1e-6, 1e-6), (1e-6, 1.0), (1.0, 1e6), (1e6, 1.0), (0.0, 1e5), (1e-3, 3e38), (1.0, 70000.0)):
        for rows in (10, 200):
            q, k, v = make(rows, 300, 4, 2, 128, torch.bfloat16)
            v = v.clamp(-1, 1)
            v[:64] *= first
            v[64:] *= rest
            got = nv.prompt_attention(q, k, v, 0.1)
            want, bound = expected(q, k, v, 0.1, [rows], [300])
            assert ((got.double() - want).abs() <= bound).all(), (first, rest)


def test_weights_of_eleven_bits():
    """Values of both signs, nearly even weights: results are small beside the values, and so is their rounding beside one of the weights to eight bits."""
    for dim, rows, length in ((128, 1, 700), (64, 150, 300), (96, 40, 40)):
        q, k, v = make(rows, length, 4, 1, dim, torch.bfloat16)
        q = q * 0.1
        got = nv.prompt_attention(q, k, v, dim ** -0.5).double()
        want, _ = expected(q, k, v, dim ** -0.5, [rows], [length])
        # errors of eleven bits are an eighth of those of eight, and add up like the values: against the rounding of the result itself
        exact = want.to(torch.bfloat16).double()
        assert (got - want).square().mean().sqrt() <= 1.05 * (exact - want).square().mean().sqrt()


def test_captured_calls_follow_their_starts():
    """Two graphs of one shape, whose starts change between the replays, from one split to several, other work between them."""
    q, k, v = make(300, 5000, 8, 2, 128, torch.bfloat16)
    starts, key_starts = ints([0, 1, 2]), ints([0, 9, 20])
    run = lambda out: nv.prompt_attention(q, k, v, 0.1, starts, key_starts, out=out)
    outs = [torch.zeros_like(q) for _ in range(3)]
    run(outs[2])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            run(out)
    for rows, lengths in (([200, 40], [300, 40]), ([1, 259], [4096, 900]), ([0, 255], [256, 4000]), ([33, 2], [33, 2]), ([260, 0], [5000, 0]), ([1, 1], [1, 4900])):
        starts.copy_(ints(starts_of(rows)))
        key_starts.copy_(ints(starts_of(lengths)))
        q.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        n = sum(rows)
        run(outs[2])
        assert torch.equal(outs[0][:n], outs[2][:n]) and torch.equal(outs[1][:n], outs[2][:n])
        want, bound = expected(q, k, v, 0.1, rows, lengths)
        assert ((outs[2].double() - want).abs() <= bound)[:n].all()


@pytest.mark.parametrize("dtype", TYPES)
def test_results_in_place_of_the_queries(dtype):
    for rows, lengths in (([150, 1, 70], [150, 1, 70]), ([20], [3000]), ([130], [0])):
        q, k, v = make(sum(rows), sum(lengths), 6, 2, 128, dtype)
        starts = ints(starts_of(rows)), ints(starts_of(lengths))
        want = nv.prompt_attention(q, k, v, 0.1, *starts)
        assert nv.prompt_attention(q, k, v, 0.1, *starts, out=q) is q and torch.equal(q, want)


def test_starts_that_are_not_ascending_stay_in_the_workspace():
    """Sequences that cover the same rows again and again, split over their keys: more states than the workspace has room for."""
    rows, keys, sequences = 300, 5000, 41
    q, k, v = make(rows, keys, 8, 2, 128, torch.bfloat16)
    starts, key_starts = (ints([n * (i % 2) for i in range(sequences + 1)]) for n in (rows, keys))
    d = _lib.PromptAttentionDescC(_lib.BF16, 128, rows, keys, 8, 2, sequences)
    for i in range(2):
        d.q_strides[i], d.k_strides[i], d.v_strides[i], d.out_strides[i] = q.stride(i), k.stride(i), v.stride(i), q.stride(i)
    d.causal, d.scale = 1, 0.1
    lib = _lib.load()
    need = lib.nvq_prompt_attention_workspace_bytes(C.byref(d))
    room = torch.full((need + (64 << 20),), 77, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    p = lambda t: C.c_void_p(t.data_ptr())
    _lib.check(lib.nvq_prompt_attention(C.byref(d), p(q), p(k), p(v), p(starts), p(key_starts), None, p(out), p(room), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    assert need > 0 and (room[need:] == 77).all()


def test_two_streams_at_once():
    sets = [make(150, 3000, 16, 4, 128, torch.bfloat16, seed=i) for i in range(2)]
    want = [nv.prompt_attention(*s, 0.1) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(nv.prompt_attention(*sets[i], 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 96), (torch.float32, 72), (torch.float16, 200)])
def test_keys_as_far_apart_as_they_may_be(dtype, dim):
    """2^24 - 8 values between two keys: offsets within a tile need all of 32 bits."""
    keys, step = 70, (1 << 24) - 8
    room = torch.empty(keys * step, device="cuda", dtype=dtype)
    q, k, v = make(30, keys, 4, 2, dim, dtype)
    far = [room[1000 * i:].as_strided(t.shape, (step, dim, 1)).copy_(t) for i, t in enumerate((k, v))]
    assert torch.equal(nv.prompt_attention(q, *far, 0.1), nv.prompt_attention(q, k, v, 0.1))
    one = [room.as_strided((1, 2, dim), (1 << 30, dim, 1)) for _ in range(2)]  # (a single key may be as far from the next as it likes)
    assert torch.equal(nv.prompt_attention(q[:1], *one, 0.1), nv.prompt_attention(q[:1], *(t.contiguous() for t in one), 0.1))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_without_end_in_shared_keys(dtype):
    """Few rows over many keys, which several blocks share: one of them meets values that are not finite, seen by some rows alone."""
    rows, length = 12, 4000
    q, k, v = make(rows, length, 4, 1, 128, dtype)
    plain = nv.prompt_attention(q, k, v, 0.05, window=3000)
    v[-5, 0, 7], v[990, 0, 3], v[2000, 0, 9] = float("inf"), float("nan"), float("-inf")
    got = nv.prompt_attention(q, k, v, 0.05, window=3000)
    # row i sees the keys 989 + i to 3988 + i
    last = length - rows + torch.arange(rows, device="cuda")
    sees = {7: last >= length - 5, 3: (last >= 990) & (last - 3000 < 990), 9: last >= 2000}
    for column, value in ((7, float("inf")), (3, float("nan")), (9, float("-inf"))):
        of = got[..., column]
        is_it = of.isnan() if value != value else of == value
        assert torch.equal(is_it, sees[column][:, None].expand_as(is_it))
    rest = torch.ones_like(got, dtype=torch.bool)
    for column, seen in sees.items():
        rest[..., column] &= ~seen[:, None]
    clean = v.clone()
    clean[-5, 0, 7], clean[990, 0, 3], clean[2000, 0, 9] = 0, 0, 0
    want, bound = expected(q, k, clean, 0.05, [rows], [length], window=3000)
    assert ((got.double() - want).abs() <= bound)[rest].all() and plain.isfinite().all()


def test_offsets_beyond_32_bits():
    """Rows so far apart that the last ones lie beyond 2^32 values."""
    rows, step = 1100, 1 << 22
    room = torch.empty(rows * step, device="cuda", dtype=torch.float16)
    apart = lambda at: room[at:].as_strided((rows, 2, 64), (step, 64, 1))
    q, k, v = make(rows, rows, 2, 2, 64, torch.float16)
    far = []
    for i, t in enumerate((q, k, v, q)):
        far.append(apart(128 * i).copy_(t))
    nv.prompt_attention(*far[:3], 0.1, out=far[3])
    assert torch.equal(far[3], nv.prompt_attention(q, k, v, 0.1))
