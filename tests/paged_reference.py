"""The paged cache's operators in 64 bits, and the inputs of their tests."""
from __future__ import annotations

import torch

import nuvec_amd as nv

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}               # half a step of the smallest values


def table(positions, dims, magnitude=1.0, base=10000.0, device="cuda"):
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] / base ** (torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims)
    return (magnitude * torch.stack([angle.cos(), angle.sin()], -1)).float()


def turned(x, angles, interleaved):
    """float64 heads `x` [..., dim] by `angles` [..., pairs, 2], and the sum of the sizes of the terms of each value."""
    c, n, pairs = angles[..., 0].double(), angles[..., 1].double(), angles.shape[-2]
    y, size = x.clone(), x.abs()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * n, b * c + a * n
    size[..., first], size[..., second] = (a * c).abs() + (b * n).abs(), (b * c).abs() + (a * n).abs()
    return y, size


def normed(x, weight, eps):
    return x.double() if weight is None else x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def codes_of(q):
    """The codes of a `Quantized` as float64, [..., dim]."""
    bits = q.quant.bits
    words = q.weight.view(torch.int32).long() & 0xFFFFFFFF
    return torch.stack([(words >> (bits * i)) & ((1 << bits) - 1) for i in range(32 // bits)], -1).flatten(-2).double()


def wide(t, group):
    return t.double().repeat_interleave(group, -1)


def random_cache(pages, key_heads, page, dim, quant, dtype, seed=0):
    """A pool of random values, quantized by `quantize`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    put = lambda: nv.quantize(torch.randn(pages, key_heads, page, dim, generator=g, device="cuda").to(dtype), quant)
    return nv.PagedCache(put(), put())


def dense(q, page_table, b, length):
    """Sequence b's rows: values [heads, length, dim], scale x (code - middle of the range) and the sizes behind a score's sum."""
    group, page = q.quant.group_size, q.weight.shape[2]
    ids = page_table[b, :-(-length // page)].long()
    rows = nv.Quantized(q.weight.view(torch.int32)[ids].view(torch.uint32), q.scales[ids], q.biases[ids], q.quant)
    c, s, z = codes_of(rows), wide(rows.scales, group), wide(rows.biases, group)
    flat = lambda t: t.transpose(0, 1).flatten(1, 2)[:, :length]
    most = 2 ** q.quant.bits
    return flat(c * s + z), flat((s * (c - most // 2)).abs()), flat(s.abs() * 2 * most + z.abs())


def attention(q, cache, page_table, lengths, scale, starts=None, sinks=None, causal=True, window=0):
    """(result, bound) of every row in 64 bits.

    The bound: queries and codes are exact.  A weight p x scale has the element type's rounding (float32: three terms, 24 bits; float16: two,
    16 bits; bfloat16: one, 8), which its values share, so its error is at most that of sum p |scale (code - middle)|.  Scores are float32 sums
    of 64 or 128 products and their biases: 32 roundings of the sum of the products' sizes, 2^-24 each (their signs are random); an error e of the
    scores moves the result by at most 2 e max |v|.  The weighted sums likewise 64 roundings of the values' sizes.  Then the result's own rounding."""
    dtype, heads = q.dtype, q.shape[1]
    key_heads, dim = cache.keys.weight.shape[1], q.shape[2]
    rep = heads // key_heads
    term = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -8}[dtype]
    want, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths):
        at, n = (b, 1) if starts is None else (starts[b], starts[b + 1] - starts[b])
        if n == 0 or length == 0:
            continue
        k, _, k_size = dense(cache.keys, page_table, b, length)
        v, v_part, v_size = dense(cache.values, page_table, b, length)
        rows = q[at:at + n].double().permute(1, 0, 2)  # [heads, n, dim]
        of = lambda t: t.repeat_interleave(rep, 0)
        scores = scale * (rows[:, :, None] * of(k)[:, None]).sum(-1) if n * length * dim * heads < 1 << 26 else scale * rows @ of(k).transpose(1, 2)
        last = (length - n + torch.arange(n, device=q.device))[:, None] if causal else torch.full((n, 1), length - 1, device=q.device)
        key = torch.arange(length, device=q.device)
        hidden = (key > last) | ((key <= last - window) if window else torch.zeros_like(key, dtype=torch.bool))
        scores = scores.masked_fill(hidden, float("-inf"))
        if sinks is not None:
            scores = torch.cat([scores, sinks.double()[:, None, None].expand(heads, n, 1)], -1)
        p = torch.softmax(scores, -1)[..., :length].nan_to_num(0.0)
        y = (p @ of(v)).permute(1, 0, 2)
        e = 32 * 2.0 ** -24 * scale * (rows.abs() @ of(k_size).transpose(1, 2)).masked_fill(hidden, 0.0).amax(-1)  # [heads, n]
        most = of(v).abs().amax((1, 2))[:, None]
        slack = (2 * e * most + 64 * 2.0 ** -24 * of(v_size).amax((1, 2))[:, None]).T[..., None]
        want[at:at + n] = y
        bound[at:at + n] = term * (p @ of(v_part)).permute(1, 0, 2) + slack + HALF[dtype] * y.abs() + TINY[dtype]
    return want, bound
