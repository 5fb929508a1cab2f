"""Attention of whole prompts (csrc/prompt_kernel.h): what a row does not see, small weights and nearly cancelling values, against 64 bits, line by line."""
import pytest
import torch

import nuvec_amd as nv
from tests.paged_reference import HALF, TINY

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TERM = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 0.0}  # what two terms of a weight leave of it


def expected(q, k, v, scale, sinks=None, causal=True, window=0):
    """(result, bound) of one sequence in 64 bits, the bound of each line from what that line sees alone.

    A weight's exponent is off by the score's float32 sum (dim roundings of 2^-24 of the sum of its terms' sizes) and by four roundings of the score, the
    weight itself by an exponential (2^-22) and its terms; an error of d in the weights moves the result by d (size + |result|), size being the weighted sum of
    the values' sizes.  The weighted sums take a rounding of 2^-24 for every product of 16 keys and of either term (float32: of two keys), the weights' sum
    one a key within a tile and one a tile.  A float16 weight below float16's normal range is off by half of its smallest step, 2^-25, where the largest of
    its tile is 2^-4 or more: by 2^-21 of the largest weight among the 64 keys on either side.  Then the result's own rounding."""
    dtype, (n, heads, dim), length, rep = q.dtype, q.shape, k.shape[0], q.shape[1] // k.shape[1]
    want, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    step = 2.0 ** -24
    last = (length - n + torch.arange(n, device=q.device))[:, None] if causal else torch.full((n, 1), length - 1, device=q.device)
    key = torch.arange(length, device=q.device)
    hidden = (key > last) | (key <= last - window) if window else key > last
    some = max(1, (1 << 25) // (n * length))
    for h in (range(i, min(i + some, j + rep)) for j in range(0, heads, rep) for i in range(j, j + rep, some)):  # heads of one key head
        h, keys, values = list(h), k[:, h[0] // rep].double(), v[:, h[0] // rep].double()
        x = q[:, h].double().transpose(0, 1)
        score = scale * x @ keys.T  # [heads, n, length]
        sizes = (abs(scale) * x.abs() @ keys.abs().T).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        score = score.masked_fill(hidden, float("-inf"))
        if sinks is not None:
            score = torch.cat([score, sinks[h].double()[:, None, None].expand(-1, n, 1)], -1)
        p = torch.softmax(score, -1)[..., :length].nan_to_num(0.0)
        y, size = p @ values, p @ values.abs()
        off = 2 * (dim + 4) * step * sizes * size + (TERM[dtype] + 2.0 ** -21 + length * (1 / 2 if dtype == torch.float32 else 1 / 8) * step) * size
        off = off + (2.0 ** -21 + (length / 32 + 64) * step + HALF[dtype]) * y.abs() + TINY[dtype]
        if dtype == torch.float16:
            near = torch.nn.functional.max_pool1d(p.float(), 129, 1, 64).double() if length > 1 else p
            off = off + 2.0 ** -21 * near @ values.abs()
        want[:, h], bound[:, h] = y.transpose(0, 1), off.transpose(0, 1)
    return want, bound


def make(rows, keys, heads, key_heads, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    put = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    return put(rows, heads, dim), put(keys, key_heads, dim), put(keys, key_heads, dim)


def within(got, want, bound, what=None):
    off = (got.double() - want).abs()
    assert got.isfinite().all() and (off <= bound).all(), (what, (off / bound).max().item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_finite_values_that_a_row_does_not_see(dtype, dim):
    """The type's large values at keys behind a row and outside its window, in a block's first tile and in later ones."""
    length = 230
    q, k, v = make(length, length, 4, 2, dim, dtype)
    for window in (0, 40):
        for large in ((1e4, 60000.0) if dtype == torch.float16 else (1e5, 1e30, -3e38)):
            for bad in (1, 60, 100, 200):
                values = v.clone()
                values[bad, :, ::3] = large
                got = nv.prompt_attention(q, k, values, 0.1, window=window)
                clean = v.clone()
                clean[bad] = 0
                blind = torch.arange(length, device="cuda") < bad
                if window:
                    blind |= torch.arange(length, device="cuda") >= bad + window
                want, bound = expected(q, k, clean, 0.1, window=window)
                within(got[blind], want[blind], bound[blind], (window, large, bad))
                want, bound = expected(q, k, values, 0.1, window=window)
                within(got, want, bound, (window, large, bad, "seen"))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_values_of_keys_that_blocks_share(dtype):
    """Few rows over many keys: a large value in one of the blocks' shares, behind some of the rows."""
    rows, length = 20, 3000
    q, k, v = make(rows, length, 4, 1, 128, dtype)
    for large in ((60000.0,) if dtype == torch.float16 else (1e30, 3e38)):
        values = v.clone()
        values[-9] = large
        got = nv.prompt_attention(q, k, values, 0.1)
        want, bound = expected(q, k, values, 0.1)
        within(got, want, bound, large)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sums_of_the_largest_values(dtype):
    """Means of values close to the type's largest, whose sums leave float32."""
    for rows, length in ((150, 150), (5, 2000)):
        q, k, v = make(rows, length, 4, 2, 128, dtype)
        v = (3e38 + 2e37 * v.float().tanh()).to(dtype)
        for sinks in (None, torch.tensor([1.0, -2.0, 3.0, 30.0], device="cuda").to(dtype)):
            got = nv.prompt_attention(q, k, v, 0.3, sinks=sinks)
            want, bound = expected(q, k, v, 0.3, sinks)
            within(got, want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_that_cancel(dtype, dim):
    """A first value that takes the others' weighted sum away but for its own rounding: what the terms of the weights leave is what remains."""
    heads = 32
    g = torch.Generator(device="cuda").manual_seed(dim)
    for length in (6, 70):
        q, k = torch.zeros(1, heads, dim, device="cuda"), torch.zeros(length, heads, dim, device="cuda")
        q[..., 0] = 1.0
        k[..., 0] = 0.7 * torch.randn(length, heads, generator=g, device="cuda")
        q, k = q.to(dtype), k.to(dtype)
        p = torch.softmax(k[..., 0].double(), 0)
        v = torch.randn(length, heads, dim, generator=g, device="cuda").to(dtype).double()
        v[0] = -(p[1:, :, None] * v[1:]).sum(0) / p[0, :, None]
        v = v.to(dtype)
        got = nv.prompt_attention(q, k, v, 1.0)
        want, bound = expected(q, k, v, 1.0)
        within(got, want, bound, length)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("length", [4000, 131073])
def test_many_small_weights(dtype, dim, length):
    many_small_weights(dtype, dim, length)


def many_small_weights(dtype, dim, length, apart=0, spread=0.3):
    """One key, of value 0, that takes nearly all of the weight, first, in the middle or last: the result is the others' alone.  (More heads than the chip has
    places for blocks, so that no block has a part of the keys; all share their keys and values.)  `apart`: a second key like it that far behind."""
    heads = 800
    g = torch.Generator(device="cuda").manual_seed(length + dim)
    put = lambda *s: torch.randn(s, generator=g, device="cuda")
    for heavy in (0, length // 2, length - 1 - apart):
        q, k, v = spread * put(1, heads, dim), spread * put(length, 1, dim), 1 + 0.25 * put(length, 1, dim)
        # (from a half of the weight to all but 6e-6 of it)
        share = torch.linspace(0.0, 12.0, heads, device="cuda")
        q[0, :, 0] = (share + torch.log(torch.tensor(float(length)))) / 8
        heavy = [heavy, heavy + apart]
        k[:, 0, 0], k[heavy, 0], v[heavy] = 0.0, 0.0, 0.0
        k[heavy, 0, 0] = 8.0
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        got = nv.prompt_attention(q, k.expand(-1, heads, -1), v.expand(-1, heads, -1), 1.0)
        want, bound = expected(q, k, v, 1.0)
        within(got, want, bound, heavy)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [4000, 131073])
def test_many_small_weights_in_float16(dim, length):
    many_small_weights(torch.float16, dim, length)


@pytest.mark.parametrize("dtype", TYPES)
def test_sums_of_many_small_weights(dtype):
    """Two keys that take nearly all of the weight, in either half of the keys that a line's two lanes add up: the others count beside both."""
    many_small_weights(dtype, 64, (1 << 19) + 1, apart=4, spread=0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads,window", [(300, 8, 0), (300, 8, 500), (3, 800, 0), (3, 2, 0)])
def test_weights_that_rise_and_fall(dtype, rows, heads, window):
    """Stretches of keys whose scores lie up to 24 apart, in any order; those of the upper ones have values of 0, so that the result is the others'."""
    length, dim = 3000, 64
    g = torch.Generator(device="cuda").manual_seed(rows + heads + window)
    put = lambda *s: torch.randn(s, generator=g, device="cuda")
    level = (24 * torch.rand(length // 50 + 1, generator=g, device="cuda")).repeat_interleave(torch.randint(1, 120, (length // 50 + 1,), generator=g, device="cuda"))
    level = torch.cat([level, torch.zeros(length, device="cuda")])[:length]
    q, k, v = 0.3 * put(rows, heads, dim), 0.3 * put(length, 1, dim), 1 + 0.25 * put(length, 1, dim)
    q[..., 0] = torch.linspace(0.2, 1.0, heads, device="cuda")
    k[:, 0, 0] = level
    v[level > 4] = 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    sinks = torch.linspace(-5.0, 30.0, heads, device="cuda").to(dtype)
    for s in (None, sinks):
        got = nv.prompt_attention(q, k.expand(-1, heads, -1), v.expand(-1, heads, -1), 1.0, sinks=s, window=window)
        want, bound = expected(q, k, v, 1.0, s, window=window)
        within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [20, 24, 25, 26, 27, 28, 30])
def test_scores_far_from_zero(dtype, power):
    """Scores that are multiples of a step of float32 near 2^power: no sum with a maximum may round a weight out of its type's range."""
    step, heads, dim = 2.0 ** (power - 23), 4, 64
    for length, rows in ((40, 1), (300, 1), (5000, 1), (300, 90)):
        place = torch.randperm(length, generator=torch.Generator().manual_seed(power + length)).to("cuda").double()
        q, k = torch.zeros(rows, heads, dim, device="cuda"), torch.zeros(length, 1, dim, device="cuda")
        _, _, v = make(1, length, 1, 1, dim, dtype)
        # score = 2^power + step x place, in parts that every type holds; log2 e times this scale is 1 in float32, so that scores and their distances are exact
        q[..., 0], k[..., 0], q[..., 1:4] = 2.0 ** (power // 2), 2.0 ** (power - power // 2), step
        k[:, 0, 1], k[:, 0, 2], k[:, 0, 3] = place % 64, place // 64 % 64 * 64, place // 4096 * 4096
        assert all(torch.equal(t, t.to(dtype).float()) for t in (q, k))
        got = nv.prompt_attention(q.to(dtype), k.to(dtype), v, 0.6931471805599453, causal=False).double()
        p = torch.exp2(step * (place - place.max()))
        p, values = p / p.sum(), v[:, 0].double()
        y, size = p @ values, p @ values.abs()
        bound = (TERM[dtype] + 2.0 ** -20) * size + (2.0 ** -20 + HALF[dtype]) * y.abs() + TINY[dtype]
        assert got.isfinite().all() and ((got - y).abs() <= bound).all(), (length, rows, ((got - y).abs() / bound).max().item())
