"""Heads between a model's projections and its attention, and the attention over a paged, quantized key / value cache.

    rotation = Rotation.new(128, 32768, base=500000.0)               # angles of 32768 positions, made once
    cache = PagedCache.new(pages=4096, key_heads=8, page_size=64, head_dim=128)
    q = append_paged(cache, k, v, page_table, positions, sequences, rotation, q=q)
    y = paged_attention(q, cache, page_table, lengths, 128 ** -0.5)  # one row per sequence

A pool's pages are shared by all sequences: position p of sequence b lies in page `page_table[b, p // page_size]`.  Page tables, positions
and lengths stay on the device and may change between replays of a captured graph.  All of it computes in libnuvec_hip.so.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .ops import _CODE, _FLOATS, InvalidArgument, Quant, QuantMode, Quantized, Unsupported, _init, _name, _ptr, _stream, _u32


# ── rotary positions ────────────────────────────────────────────────────────────────────────────────────────────────
def rotation_freqs(dims: int, base: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[Optional[torch.Tensor], float, float]:
    """`(freqs, scale, magnitude)` for `Rotation.new` from a checkpoint's `rope_scaling` entry: none, "linear" (positions divided by
    `factor`), "llama3" (long waves slowed by `factor`, short ones kept, a blend between) or "yarn" (the same by the number of turns, with a
    magnitude; the blend begins and ends at whole pairs unless `truncate` is false).  `freqs` is None or float64 `[dims / 2]`: the values that positions are divided by."""
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return None, 1.0, 1.0
    if dims <= 0 or dims % 2:
        raise InvalidArgument(f"rotation_freqs: {dims} rotary values")
    if kind not in ("linear", "llama3", "yarn"):
        raise Unsupported(f"rotation_freqs: scaling '{kind}'")

    def number(key: str, otherwise: Optional[float] = None) -> float:
        value = scaling.get(key)
        if value is None and otherwise is None:
            raise InvalidArgument(f"rotation_freqs: scaling '{kind}' without {key}")
        return float(otherwise if value is None else value)

    factor = number("factor")
    if kind == "linear":
        return None, 1.0 / factor, 1.0
    freqs = base ** (torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if kind == "llama3":
        low, high = number("low_freq_factor"), number("high_freq_factor")
        turns = number("original_max_position_embeddings") / (2 * math.pi * freqs)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return 1.0 / ((1.0 - keep) / (factor * freqs) + keep / freqs), 1.0, 1.0
    most = number("original_max_position_embeddings")
    at = lambda turns: dims * math.log(most / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = at(number("beta_fast", 32.0)), at(number("beta_slow", 1.0))
    if scaling.get("truncate") in (None, True):  # (the blend begins and ends at whole pairs)
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dims - 1)
    slowed = ((torch.arange(dims // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    magnitude = lambda m: 1.0 if factor <= 1.0 else 0.1 * m * math.log(factor) + 1.0
    magnitudes = magnitude(number("mscale", 1.0)) / magnitude(number("mscale_all_dim", 0.0))
    return 1.0 / (slowed / (factor * freqs) + (1.0 - slowed) / freqs), 1.0, number("attention_factor", magnitudes)


@dataclass
class Rotation:
    """The angles of positions 0 .. positions - 1, float32 `[positions, dims / 2, 2]` (cosine, sine), and which values of a head pair up:
    `(i, i + dims / 2)` or, `interleaved`, `(2 i, 2 i + 1)`, of its first `dims` values."""
    table: torch.Tensor
    interleaved: bool = False

    @property
    def dims(self) -> int:
        return 2 * self.table.shape[1]

    @staticmethod
    def new(dims: int, positions: int, base: float = 10000.0, scale: float = 1.0, interleaved: bool = False,
            freqs: Optional[torch.Tensor] = None, magnitude: float = 1.0, device="cuda") -> "Rotation":
        """Angles `scale * position / freqs[i]` in 64 bits, freqs `base^(2 i / dims)` unless given (float64, or float32 values); cosines and sines
        times `magnitude`, rounded once."""
        if dims <= 0 or dims % 2 or positions < 1:
            raise InvalidArgument(f"rotation: {dims} values, {positions} positions")
        table = torch.empty((positions, dims // 2, 2), dtype=torch.float32, device=device)
        _init(table)
        if freqs is not None:
            if tuple(freqs.shape) != (dims // 2,):
                raise InvalidArgument(f"rotation: freqs {list(freqs.shape)} for {dims} values")
            freqs = freqs.to(device=table.device, dtype=torch.float64 if freqs.dtype == torch.float64 else torch.float32).contiguous()
        lib = _lib.load()
        make = lib.nvq_rotation_table_f64 if freqs is not None and freqs.dtype == torch.float64 else lib.nvq_rotation_table
        _lib.check(make(_ptr(freqs), dims, positions, float(base), float(scale), float(magnitude), _ptr(table), _stream()))
        return Rotation(table, interleaved)


def _same_device(op: str, x: torch.Tensor, *others) -> None:
    for t in others:
        if t is not None and t.device != x.device:
            raise InvalidArgument(f"{op}: operands on {x.device} and {t.device}")


def _angles(op: str, rotation: Optional[Rotation], dim: int, x: torch.Tensor):
    """The rotation's table, rotary values, interleaving and positions."""
    if rotation is None:
        return None, 0, 0, 0
    t = rotation.table
    if t.dtype != torch.float32 or t.ndim != 3 or t.shape[2] != 2 or t.shape[0] < 1 or not t.is_contiguous():
        raise InvalidArgument(f"{op}: the table of angles must be float32 [positions, pairs, 2], got {_name(t.dtype)} {list(t.shape)}")
    if rotation.dims > dim:
        raise InvalidArgument(f"{op}: {rotation.dims} rotary values of heads of {dim}")
    _same_device(op, x, t)
    return t, rotation.dims, int(rotation.interleaved), t.shape[0]


def _weight(op: str, w: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.dtype != x.dtype or tuple(w.shape) != (x.shape[-1],):
        raise InvalidArgument(f"{op}: a norm's weight must be {_name(x.dtype)} [{x.shape[-1]}], got {_name(w.dtype)} {list(w.shape)}")
    _same_device(op, x, w)
    return w.contiguous()


def _indices(op: str, what: str, t: torch.Tensor, shape, x: torch.Tensor) -> torch.Tensor:
    """int32 `t` of `shape`, contiguous."""
    if t.dtype != torch.int32 or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise InvalidArgument(f"{op}: {what} must be int32 {'' if shape is None else list(shape)}, got {_name(t.dtype)} {list(t.shape)}")
    _same_device(op, x, t)
    return t.contiguous()


def _heads(op: str, x: torch.Tensor) -> torch.Tensor:
    if x.dtype not in _FLOATS:
        raise InvalidArgument(f"{op}: unsupported dtype {_name(x.dtype)}")
    if x.ndim != 4:
        raise InvalidArgument(f"{op}: heads must be [batch, heads, length, dim], got {list(x.shape)}")
    if not 1 <= x.shape[3] <= 512:
        raise Unsupported(f"{op}: heads of {x.shape[3]} values (512 at most)")
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def _own_rows(op: str, out: torch.Tensor) -> None:
    """An expanded output would be written by several rows at once."""
    if any(n > 1 and step == 0 for n, step in zip(out.shape, out.stride())):
        raise InvalidArgument(f"{op}: rows of the output {list(out.shape)} share their memory")


def _out_like(op: str, x: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    if out is None:
        y = torch.empty_like(x)  # (the strides' order is x's; one of overlapping rows may put another dimension innermost)
        return y if y.stride(3) == 1 or x.shape[3] == 1 else torch.empty_like(x, memory_format=torch.contiguous_format)
    if out.dtype != x.dtype or out.shape != x.shape or (out.numel() > 0 and out.stride(-1) != 1 and out.shape[-1] != 1):
        raise InvalidArgument(f"{op}: the output must be {_name(x.dtype)} {list(x.shape)} with consecutive values")
    _own_rows(op, out)
    _same_device(op, x, out)
    return out


def _rotate(op: str, xs, weights, outs, rotation, offset, eps):
    x = xs[0]
    b, _, l, d = x.shape
    table, dims, interleaved, rows = _angles(op, rotation, d, x)
    desc = _lib.HeadRopeDescC(_CODE[x.dtype], d, dims, interleaved, 0, rows, b, l)
    offsets = None
    if isinstance(offset, torch.Tensor):
        if offset.ndim not in (1, 2):
            raise InvalidArgument(f"{op}: offsets must be [batch] or [batch, length], got {list(offset.shape)}")
        offsets = _indices(op, "offsets", offset, (b,) if offset.ndim == 1 else (b, l), x)
        desc.per_position = int(offset.ndim == 2)
    else:
        if rotation is not None and (offset < 0 or offset + l > rows):
            raise InvalidArgument(f"{op}: positions {offset} to {offset + l - 1} of a table of {rows}")
        desc.offset = offset
    desc.eps = eps
    ys = []
    for i, (t, out) in enumerate(zip(xs, outs)):
        y = _out_like(op, t, out)
        desc.heads[i] = t.shape[1]
        for k in range(3):
            desc.x_strides[i][k], desc.y_strides[i][k] = t.stride(k), y.stride(k)
        ys.append(y)
    _init(x)
    p = [_ptr(v) for t, w, y in zip(xs, weights, ys) for v in (t, w, y)] + [C.c_void_p(None)] * (6 - 3 * len(xs))
    _lib.check(_lib.load().nvq_head_norm_rope(C.byref(desc), _ptr(table), _ptr(offsets), *p, _stream()))
    return ys


def rope(x: torch.Tensor, rotation: Rotation, offset: Union[int, torch.Tensor] = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions of `x` `[batch, heads, length, dim]` (any strides with consecutive values of a head; MLX's `fast.rope`): the first
    `rotation.dims` values of a head turn, the others stay.  Element l is at position `offset + l`; `offset` is an int, int32 `[batch]`, or int32
    `[batch, length]` for positions one by one.  Positions on the device outside the table are clamped to it.  `out` may be `x` itself, unless rows of it share their memory."""
    y = (_lib._native or _lib.native()).rope(x, rotation, offset, out)
    if y is not None:
        return y if out is None else out
    return _rotate("rope", (_heads("rope", x),), (None,), (out,), rotation, offset, 0.0)[0]


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   rotation: Optional[Rotation] = None, offset: Union[int, torch.Tensor] = 0, eps: float = 1e-6):
    """The RMS norms over each head of queries and keys (`[batch, heads, length, dim]`, their own numbers of heads; weights `[dim]`, None: not
    normed) and their rotation, in one pass over both: `(q, k)`, rounded once.  `offset` as in `rope`."""
    done = (_lib._native or _lib.native()).head_norm_rope(q, k, q_weight, k_weight, rotation, offset, eps)
    if done is not None:
        return done
    op = "head_norm_rope"
    q, k = _heads(op, q), _heads(op, k)
    if k.dtype != q.dtype or (k.shape[0], k.shape[2], k.shape[3]) != (q.shape[0], q.shape[2], q.shape[3]):
        raise InvalidArgument(f"{op}: queries {_name(q.dtype)} {list(q.shape)} and keys {_name(k.dtype)} {list(k.shape)}")
    _same_device(op, q, k)
    return tuple(_rotate(op, (q, k), (_weight(op, q_weight, q), _weight(op, k_weight, k)), (None, None), rotation, offset, eps))


# ── the paged cache ─────────────────────────────────────────────────────────────────────────────────────────────────
@dataclass
class PagedCache:
    """Keys and values of many sequences in pages of a pool: `Quantized` affine codes `[pages, key_heads, page_size, dim * bits / 32]`, scales and
    biases `[pages, key_heads, page_size, dim / group]`.  4 and 8 bits, heads of 64 and 128 values, pages of a power of two of 16 to 1024
    positions.  (`dequantize` of either gives its pages as values.)"""
    keys: Quantized
    values: Quantized

    @staticmethod
    def new(pages: int, key_heads: int, page_size: int, head_dim: int, quant: Quant = Quant(), dtype: torch.dtype = torch.bfloat16,
            device="cuda") -> "PagedCache":
        """An empty pool (zeros)."""
        group, bits = quant.checked("paged_cache")
        if quant.mode != QuantMode.AFFINE or dtype not in _FLOATS or head_dim % group:
            raise InvalidArgument(f"paged_cache: {quant.mode.mlx_name} groups of {group} of heads of {head_dim}, {_name(dtype)}")
        shape = (pages, key_heads, page_size)
        zeros = lambda last, t: torch.zeros(shape + (last,), dtype=t, device=device)
        of = lambda: Quantized(_u32(zeros(head_dim * bits // 32, torch.int32)), zeros(head_dim // group, dtype), zeros(head_dim // group, dtype), quant)
        return PagedCache(of(), of())

    @property
    def page_size(self) -> int:
        return self.keys.weight.shape[2]

    @property
    def key_heads(self) -> int:
        return self.keys.weight.shape[1]


def _paged(op: str, cache: PagedCache, dim: Optional[int], dtype: Optional[torch.dtype], page_table: torch.Tensor):
    """The cache's descriptor and tensors."""
    k, v = cache.keys, cache.values
    if k.quant != v.quant or k.quant.mode != QuantMode.AFFINE or k.biases is None or v.biases is None:
        raise InvalidArgument(f"{op}: keys and values need one affine quantization")
    group, bits = k.quant.checked(op)
    w = _u32(k.weight)
    if w.ndim != 4:
        raise InvalidArgument(f"{op}: pages must be [pages, key heads, page, words], got {list(w.shape)}")
    d = w.shape[3] * 32 // bits
    if d % group or w.shape[3] * 32 != d * bits:
        raise InvalidArgument(f"{op}: {w.shape[3]} words are no groups of {group} values of {bits} bits")
    scales = tuple(w.shape[:3]) + (d // group,)
    kind = k.scales.dtype if dtype is None else dtype
    for q in (k, v):
        if _u32(q.weight).dtype != torch.uint32 or q.weight.shape != w.shape or tuple(q.scales.shape) != scales or tuple(q.biases.shape) != scales \
                or q.scales.dtype != kind or q.biases.dtype != kind:
            raise InvalidArgument(f"{op}: codes {list(q.weight.shape)}, scales {_name(q.scales.dtype)} {list(q.scales.shape)} of a cache of {_name(kind)} {list(w.shape)}")
        if not (q.weight.is_contiguous() and q.scales.is_contiguous() and q.biases.is_contiguous()):
            raise InvalidArgument(f"{op}: a cache's pages must be contiguous")
        _same_device(op, w, q.weight, q.scales, q.biases)
    if dim is not None and dim != d:
        raise InvalidArgument(f"{op}: heads of {dim} values over a cache of {d}")
    if kind not in _FLOATS:
        raise InvalidArgument(f"{op}: unsupported dtype {_name(kind)}")
    if page_table.dtype != torch.int32 or page_table.ndim != 2:
        raise InvalidArgument(f"{op}: the page table must be int32 [sequences, columns], got {_name(page_table.dtype)} {list(page_table.shape)}")
    _same_device(op, w, page_table)
    if page_table.numel() > 0 and (page_table.stride(1) != 1 or page_table.stride(0) < page_table.shape[1]):
        page_table = page_table.contiguous()
    desc = _lib.PagedDescC(_CODE[kind], bits, group, d, w.shape[0], w.shape[2], w.shape[1], page_table.shape[0], page_table.shape[1],
                           max(page_table.stride(0), page_table.shape[1]))
    return desc, page_table, (w, k.scales, k.biases, _u32(v.weight), v.scales, v.biases)


def _rows(op: str, what: str, x: torch.Tensor, heads: Optional[int], like: torch.Tensor) -> torch.Tensor:
    """`[tokens, heads, dim]` beside the keys (or queries) `like`, values of a head consecutive."""
    if x.ndim != 3 or x.dtype != like.dtype or x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2] or (heads is not None and x.shape[1] != heads):
        raise InvalidArgument(f"{op}: {what} {_name(x.dtype)} {list(x.shape)} beside {_name(like.dtype)} {list(like.shape)}")
    _same_device(op, like, x)
    return x if x.stride(2) == 1 else x.contiguous()


def append_paged(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, positions: torch.Tensor,
                 sequences: Optional[torch.Tensor] = None, rotation: Optional[Rotation] = None, k_weight: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
    """Writes token t's keys and values (`[tokens, key_heads, dim]`) to position `positions[t]` of sequence `sequences[t]` (int32; None: t) of the
    cache: the keys normed (`k_weight`), rotated to their position and quantized from the float32 result, the values quantized.  `q` `[tokens,
    query_heads, dim]`: the same tokens' queries, normed (`q_weight`) and rotated in the same launch; they are the result (None without them).

    A token with a negative position is padding: nothing is written.  Neither is one whose position lies outside the rotation's table or the page
    table, or whose page is not in the pool.  Two tokens of one position are the caller's error.  (Codes are the nearest to the scale and bias as
    stored, those of `quantize` to the unrounded ones.)"""
    done = (_lib._native or _lib.native()).append_paged(cache, k, v, page_table, positions, sequences, rotation, k_weight, q, q_weight, eps)
    if done is not None:
        return None if done is True else done
    op = "append_paged"
    if k.ndim != 3 or k.dtype not in _FLOATS:
        raise InvalidArgument(f"{op}: keys must be [tokens, key heads, dim] of a float type, got {_name(k.dtype)} {list(k.shape)}")
    cd, page_table, pool = _paged(op, cache, k.shape[2], k.dtype, page_table)
    _same_device(op, pool[0], k)
    k = _rows(op, "keys", k, cd.key_heads, k)
    v = _rows(op, "values", v, cd.key_heads, k)
    tokens = k.shape[0]
    positions = _indices(op, "positions", positions, (tokens,), k)
    sequences = None if sequences is None else _indices(op, "sequences", sequences, (tokens,), k)
    if sequences is None and page_table.shape[0] != tokens:
        raise InvalidArgument(f"{op}: {tokens} tokens of {page_table.shape[0]} sequences without `sequences`")
    table, dims, interleaved, rows = _angles(op, rotation, k.shape[2], k)
    k_weight = _weight(op, k_weight, k)
    desc = _lib.PagedAppendDescC(cd, tokens, 0, dims, interleaved, rows)
    desc.eps = eps
    out = None
    if q is None:
        q_weight = None
    else:
        q = _rows(op, "queries", q, None, k)
        q_weight = _weight(op, q_weight, q)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        desc.query_heads = q.shape[1]
    for i in range(2):
        desc.k_strides[i], desc.v_strides[i] = k.stride(i), v.stride(i)
        if q is not None:
            desc.q_strides[i] = q.stride(i)
    _init(k)
    _lib.check(_lib.load().nvq_append_paged(C.byref(desc), _ptr(page_table), _ptr(sequences), _ptr(positions), _ptr(table), _ptr(q), _ptr(q_weight),
                                            _ptr(out), _ptr(k), _ptr(k_weight), _ptr(v), *(_ptr(t) for t in pool), _stream()))
    return out


def read_paged(cache: PagedCache, page_table: torch.Tensor, positions: torch.Tensor, sequences: Optional[torch.Tensor] = None):
    """Positions of the cache as values: `(keys, values)`, each `[tokens, key_heads, dim]` in the scales' type, code * scale + bias rounded once;
    row t is position `positions[t]` of sequence `sequences[t]` (int32; None: t), zeros where `append_paged` would write nothing."""
    done = (_lib._native or _lib.native()).read_paged(cache, page_table, positions, sequences)
    if done is not None:
        return done
    op = "read_paged"
    cd, page_table, pool = _paged(op, cache, None, None, page_table)
    if positions.ndim != 1:
        raise InvalidArgument(f"{op}: positions must be int32 [tokens], got {list(positions.shape)}")
    tokens = positions.shape[0]
    positions = _indices(op, "positions", positions, None, pool[0])
    sequences = None if sequences is None else _indices(op, "sequences", sequences, (tokens,), pool[0])
    if sequences is None and page_table.shape[0] != tokens:
        raise InvalidArgument(f"{op}: {tokens} tokens of {page_table.shape[0]} sequences without `sequences`")
    _init(pool[0])
    keys, values = (torch.empty((tokens, cd.key_heads, cd.head_dim), dtype=pool[1].dtype, device=pool[0].device) for _ in range(2))
    _lib.check(_lib.load().nvq_read_paged(C.byref(cd), tokens, _ptr(page_table), _ptr(sequences), _ptr(positions), *(_ptr(t) for t in pool), _ptr(keys),
                                          _ptr(values), _stream()))
    return keys, values


def paged_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                    query_starts: Optional[torch.Tensor] = None, max_queries: Optional[int] = None, sinks: Optional[torch.Tensor] = None,
                    causal: bool = True, window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`softmax(scale * q K^T [, sinks]) V` of the rows `q` `[rows, query_heads, dim]`, each over its sequence's positions in the cache.

    Sequence b has `lengths[b]` positions (int32 `[sequences]`), those of its own rows among them, and the rows `query_starts[b]` to
    `query_starts[b + 1] - 1` (int32 `[sequences + 1]`, ascending; None: row b alone).  With `causal` row i of n sees the positions up to
    `lengths[b] - n + i`, with `window` the last `window` of those alone.  `sinks` `[query_heads]` join each head's softmax.  Rows that see nothing are
    zeros; rows of no sequence are left as they were in `out` (and undefined in a new result).  `max_queries` is the most rows of a sequence, as
    far as the caller knows: it sizes the launch, more rows are right all the same.

    The keys' and values' codes are exact operands; the softmax's weights, times the values' scales, hold 16 bits (24 in float32), everything else is
    float32."""
    y = (_lib._native or _lib.native()).paged_attention(q, cache, page_table, lengths, scale, query_starts, max_queries, sinks, causal, window, out)
    if y is not None:
        return y if out is None else out
    op = "paged_attention"
    if q.ndim != 3 or q.dtype not in _FLOATS:
        raise InvalidArgument(f"{op}: queries must be [rows, query heads, dim] of a float type, got {_name(q.dtype)} {list(q.shape)}")
    cd, page_table, pool = _paged(op, cache, q.shape[2], q.dtype, page_table)
    _same_device(op, pool[0], q)
    q = q if q.stride(2) == 1 else q.contiguous()
    n, heads, d = q.shape
    lengths = _indices(op, "lengths", lengths, (cd.sequences,), q)
    if query_starts is None:
        if n != cd.sequences:
            raise InvalidArgument(f"{op}: {n} rows of {cd.sequences} sequences without query starts")
    else:
        query_starts = _indices(op, "query starts", query_starts, (cd.sequences + 1,), q)
    if sinks is not None:
        if sinks.dtype != q.dtype or tuple(sinks.shape) != (heads,):
            raise InvalidArgument(f"{op}: sinks must be {_name(q.dtype)} [{heads}], got {_name(sinks.dtype)} {list(sinks.shape)}")
        _same_device(op, q, sinks)
        sinks = sinks.contiguous()
    if window < 0:
        raise InvalidArgument(f"{op}: a window of {window}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or out.shape != q.shape or out.stride(2) != 1:
        raise InvalidArgument(f"{op}: the output must be {_name(q.dtype)} {list(q.shape)} with consecutive values")
    _own_rows(op, out)
    _same_device(op, q, out)
    desc = _lib.PagedAttentionDescC(cd, n, heads, 1 if query_starts is None else n if max_queries is None else max(1, min(n, int(max_queries))))
    for i in range(2):
        desc.q_strides[i], desc.out_strides[i] = q.stride(i), out.stride(i)
    desc.window, desc.causal, desc.scale = min(window, 1 << 62), int(causal), float(scale)  # (ctypes would take a larger one modulo 2^64)
    _init(q)
    lib = _lib.load()
    need = lib.nvq_paged_attention_workspace_bytes(C.byref(desc))
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.check(lib.nvq_paged_attention(C.byref(desc), _ptr(q), *(_ptr(t) for t in pool), _ptr(page_table), _ptr(lengths), _ptr(query_starts), _ptr(sinks),
                                       _ptr(out), _ptr(workspace), _stream()))
    return out
