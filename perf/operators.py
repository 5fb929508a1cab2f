"""The operators around a paged, quantized key / value cache, as cases that can be timed and compared.

A case is a dict of plain values; its `op` names the operator:

  rope        rotary positions of queries or keys (`rope`)
  norm        the norms of the queries' and keys' heads with the rotation (`head_norm_rope`)
  append      new keys, rotated (and normed), and values quantized into the pages of a cache, with the queries beside them
              (`append_paged`), and the rows read back as the values they stand for (`read_paged`)
  attention   attention over the pages, one row per sequence or ragged rows (`paged_attention`)

With `own` false `run` computes them in elementary torch operations, in 32 bits (sums of squares in 64: a code of four bits turns
over on the last bit of a norm); with `own` true it makes the package's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
DTYPE_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}
EPS = 1e-6

# The largest work of a drawn case, that of the largest listed ones: a prompt of 8192 tokens through 32 heads, the cache of 131072
# positions, and a chunk of 1024 queries of 32 heads over 4096 positions.
MOST_VALUES = 8192 * 32 * 128
MOST_TOKENS = 6000 * 48 * 128
MOST_CACHE = 131072 * 8 * 128  # (of 4 bits)
MOST_SCORES = 32 * 1024 * 4096


def listed():
    return [
        # The queries of eight requests' next tokens, each at its own position: the smallest call of a step.
        {"name": "rope_step", "op": "rope", "dtype": "bfloat16", "batch": 8, "heads": 32, "length": 1, "dim": 128, "rotary": 128,
         "interleaved": False, "scaling": "none", "table": 8192},
        # A long prompt's queries as the projection leaves them (tokens outermost), frequencies scaled for a long context.
        {"name": "rope_prompt", "op": "rope", "dtype": "bfloat16", "batch": 1, "heads": 32, "length": 8192, "dim": 128, "rotary": 128,
         "interleaved": False, "scaling": "bands", "table": 131072},
        # Interleaved pairs, a part of a head that is no power of two, ragged sizes.
        {"name": "rope_partial", "op": "rope", "dtype": "float16", "batch": 3, "heads": 13, "length": 517, "dim": 80, "rotary": 32,
         "interleaved": True, "scaling": "linear", "table": 4096},
        # A decode step's queries and keys of sixteen requests, normed and rotated.
        {"name": "norm_step", "op": "norm", "dtype": "bfloat16", "batch": 16, "heads": 32, "key_heads": 8, "length": 1, "dim": 128,
         "rotary": 128, "interleaved": False, "scaling": "none", "table": 32768},
        # Two prompts' queries and keys together.
        {"name": "norm_prompt", "op": "norm", "dtype": "bfloat16", "batch": 2, "heads": 32, "key_heads": 8, "length": 2049, "dim": 128,
         "rotary": 128, "interleaved": False, "scaling": "none", "table": 32768},
        # The step of 64 requests: norms, rotation, quantization and the queries beside them; some rows of the batch are padding.
        {"name": "append_step", "op": "append", "dtype": "bfloat16", "bits": 4, "group": 64, "dim": 128, "heads": 32, "key_heads": 8,
         "page": 16, "sequences": 64, "tokens": 64, "rotary": 128, "interleaved": False, "norm": True, "queries": True, "table": 32768},
        # Three prompts' ragged chunks in one call.
        {"name": "append_prompt", "op": "append", "dtype": "bfloat16", "bits": 4, "group": 64, "dim": 128, "heads": 32, "key_heads": 8,
         "page": 64, "sequences": 3, "tokens": 6000, "rotary": 128, "interleaved": False, "norm": False, "queries": True, "table": 32768},
        # 8-bit pages of small heads, half of each rotated, keys and values alone.
        {"name": "append_8bit", "op": "append", "dtype": "float16", "bits": 8, "group": 32, "dim": 64, "heads": 10, "key_heads": 5,
         "page": 32, "sequences": 7, "tokens": 777, "rotary": 32, "interleaved": True, "norm": False, "queries": False, "table": 8192},
        # A decode step of sixteen requests of up to 8192 positions.
        {"name": "attention_step", "op": "attention", "dtype": "bfloat16", "bits": 4, "group": 64, "dim": 128, "heads": 32,
         "key_heads": 8, "page": 64, "batch": 16, "queries": 1, "positions": 8192, "sinks": False, "window": 0},
        # One request at the end of a very long context: the work is split over its positions.
        {"name": "attention_long", "op": "attention", "dtype": "bfloat16", "bits": 4, "group": 64, "dim": 128, "heads": 32,
         "key_heads": 8, "page": 256, "batch": 1, "queries": 1, "positions": 131072, "sinks": False, "window": 0},
        # A 1024-token chunk of one prompt over 4096 positions.
        {"name": "attention_prompt", "op": "attention", "dtype": "bfloat16", "bits": 4, "group": 64, "dim": 128, "heads": 32,
         "key_heads": 8, "page": 64, "batch": 1, "queries": 1024, "positions": 4096, "sinks": False, "window": 0},
        # Chunks and single tokens in one call over 8-bit pages of small heads, with sinks and a window.
        {"name": "attention_mixed", "op": "attention", "dtype": "float16", "bits": 8, "group": 32, "dim": 64, "heads": 20,
         "key_heads": 5, "page": 32, "batch": 9, "queries": 200, "positions": 2500, "sinks": True, "window": 1000},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: its operator and formats by how often they are met, its sizes over the whole range."""
    op = rng.choice(["rope", "norm", "append", "append", "attention", "attention", "attention"])
    c = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "float16"])}
    if op in ("rope", "norm"):
        c["dtype"] = rng.choice([c["dtype"], c["dtype"], "float32"])
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        c.update(batch=_log(rng, 1, 64), heads=_log(rng, 1, 64), dim=dim, rotary=rng.choice([dim, dim, dim // 2, 2 * (dim // 5)]),
                 interleaved=rng.random() < 0.3, scaling=rng.choice(["none", "linear", "bands"]), table=rng.choice([8192, 32768, 131072]))
        if op == "norm":
            c["key_heads"] = _log(rng, 1, 16)
        most = MOST_VALUES * 2 // DTYPE_BYTES[c["dtype"]] // (c["batch"] * (c["heads"] + c.get("key_heads", 0)) * dim)
        c["length"] = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, min(8192, most)))
        return c
    dim, key_heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 5, 8, 8])
    c.update(bits=rng.choice([4, 4, 4, 8]), group=rng.choice([32, 64, 64, dim]), dim=dim, key_heads=key_heads,
             heads=key_heads * rng.choice([1, 2, 3, 4, 4, 8]), page=rng.choice([16, 32, 64, 128, 256]))
    if op == "append":
        sequences = _log(rng, 1, 128)
        c.update(sequences=sequences, rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5,
                 queries=rng.random() < 0.7, table=rng.choice([8192, 32768]))
        most = max(sequences, min(6000, MOST_TOKENS // ((c["heads"] * c["queries"] + 2 * key_heads * (2 if c["bits"] == 8 else 1)) * dim)))
        c["tokens"] = sequences if rng.random() < 0.4 else _log(rng, sequences, most)
        return c
    c.update(sinks=rng.random() < 0.3, window=rng.choice([0, 0, 0, _log(rng, 16, 2048)]))
    if rng.random() < 0.55:
        batch = _log(rng, 1, 64)
        c.update(batch=batch, queries=1, positions=_log(rng, 16, max(16, min(131072, MOST_CACHE * 4 // (c["bits"] * batch * key_heads * dim)))))
    else:
        batch, positions = _log(rng, 1, 12), _log(rng, 32, 8192)
        most = min(MOST_SCORES // (batch * positions * c["heads"]), 1024, positions)
        c.update(batch=batch, positions=positions, queries=_log(rng, 2, max(2, most)))
    return c


# ── inputs ──────────────────────────────────────────────────────────────────────────────────────────────────────────
def _table(case, device):
    """The rotation's table, as a program makes it once: cosines and sines of every position's angles, the angles in 64 bits."""
    half, base = case["rotary"] // 2, 500000.0
    inverse = base ** (-torch.arange(half, device=device, dtype=torch.float64) * 2 / case["rotary"])
    scaling = case.get("scaling", "none")
    if scaling == "linear":
        inverse = inverse / 4
    elif scaling == "bands":  # long waves slowed eightfold, short ones kept, a blend between
        wave = 2 * math.pi / inverse
        blend = ((8192 / wave - 1) / 3).clamp(0, 1)
        inverse = (1 - blend) * inverse / 8 + blend * inverse
    angle = torch.arange(case["table"], device=device, dtype=torch.float64)[:, None] * inverse
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _pool(case, pages, device):
    """The pages of keys or of values: codes, scales and biases [pages, key heads, page, ...], and one page more that no table names."""
    shape = (pages + 1, case["key_heads"], case["page"])
    dtype, groups = DTYPES[case["dtype"]], case["dim"] // case["group"]
    return {"codes": torch.zeros(shape + (case["dim"] * case["bits"] // 32,), dtype=torch.int32, device=device),
            "scales": torch.zeros(shape + (groups,), dtype=dtype, device=device), "biases": torch.zeros(shape + (groups,), dtype=dtype, device=device)}


def _handle(s, case):
    """What a program that uses the package keeps beside these tensors: its objects over them."""
    import nuvec_amd as nv
    if "table" in s:
        s["rotation"] = nv.Rotation(s["table"], case["interleaved"])
    if "keys" in s:
        of = lambda p: nv.Quantized.affine(p["codes"].view(torch.uint32), p["scales"], p["biases"], case["group"], case["bits"])
        s["cache"] = nv.PagedCache(of(s["keys"]), of(s["values"]))


def _lengths(case):
    """(new rows, positions with them) of each sequence: the first has the most positions, others down to a half; ragged batches mix
    whole chunks, single tokens and short ends, one of them with more rows than positions, one with none at all."""
    rows, positions = [], []
    for b in range(case["batch"]):
        most = case["positions"] - (b * 37 % 64) * case["positions"] // 128
        n = 1 if case["queries"] == 1 else (case["queries"], 1, max(1, case["queries"] // 7))[b % 3]
        if case["queries"] > 1 and b == 4:
            n, most = 3, 2
        elif case["queries"] > 1 and b == 7:
            n, most = 1, 0
        rows.append(n)
        positions.append(most if b in (4, 7) else max(n, most))
    return rows, positions


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    dtype, dim = DTYPES[case["dtype"]], case["dim"]
    normal = lambda *shape: torch.randn(shape, generator=g, device=device)
    s = {"case": case}
    if case["op"] in ("rope", "norm"):
        batch, length = case["batch"], case["length"]
        s["table"] = _table(case, device)
        s["offset"] = torch.randint(0, case["table"] - length + 1, (batch,), generator=g, device=device, dtype=torch.int32)
        heads = (("q", case["heads"]),) + ((("k", case["key_heads"]),) if case["op"] == "norm" else ())
        for name, h in heads:  # heads [batch, heads, length, dim] over tokens outermost, as projections leave them
            s[name] = normal(batch, length, h, dim).to(dtype).transpose(1, 2)
            s[name + "_weight"] = (1 + 0.2 * normal(dim)).to(dtype)
    elif case["op"] == "append":
        tokens, sequences, page = case["tokens"], case["sequences"], case["page"]
        each = [tokens // sequences + (i < tokens % sequences) for i in range(sequences)]
        held = [(i * 29 + 5) % (3 * page) for i in range(sequences)]  # positions that the sequences have already
        columns = max(-(-(h + n) // page) for h, n in zip(held, each))
        table = torch.randperm(sequences * columns, generator=g, device=device).to(torch.int32).reshape(sequences, columns)
        positions = torch.cat([torch.arange(h, h + n) for h, n in zip(held, each)]).to(torch.int32)
        positions[5::23] = -1  # rows of the batch that are padding
        s.update(table=_table(case, device), page_table=table, positions=positions.to(device),
                 sequences=torch.repeat_interleave(torch.arange(sequences), torch.tensor(each)).to(torch.int32).to(device))
        spread = torch.exp(0.5 * normal(case["key_heads"], dim))  # (channels of keys differ in size)
        s["k"], s["v"] = (normal(tokens, case["key_heads"], dim) * spread).to(dtype), normal(tokens, case["key_heads"], dim).to(dtype)
        s["q"] = normal(tokens, case["heads"], dim).to(dtype) if case["queries"] else None
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * normal(dim)).to(dtype) if case["norm"] else None for _ in range(2))
        s["keys"], s["values"] = (_pool(case, sequences * columns, device) for _ in range(2))
    else:
        page, (rows, positions) = case["page"], _lengths(case)
        columns = -(-max(positions) // page)
        held = [-(-n // page) for n in positions]
        ids = torch.randperm(sum(held), generator=g, device=device).to(torch.int32)
        table = torch.zeros((case["batch"], columns), dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(held):
            table[b, :n] = ids[at:at + n]
            at += n
        starts = torch.tensor([0] + rows).cumsum(0)
        s.update(page_table=table, lengths=torch.tensor(positions, dtype=torch.int32, device=device),
                 starts=None if case["queries"] == 1 else starts.to(torch.int32).to(device), scale=dim ** -0.5)
        spread = torch.exp(0.5 * normal(case["key_heads"], 1, dim))
        for name in ("keys", "values"):
            s[name] = p = _pool(case, sum(held), device)
            x = normal(sum(held), case["key_heads"], page, dim).to(dtype).float()
            codes, scales, biases = _codes(x * spread if name == "keys" else x, case)
            p["codes"][:-1], p["scales"][:-1], p["biases"][:-1] = codes, scales, biases
        s["q"] = normal(int(starts[-1]), case["heads"], dim).to(dtype)
        s["sinks"] = normal(case["heads"]).to(dtype) if case["sinks"] else None
        # which sequence a row belongs to and which of its rows it is
        s["row_sequence"] = torch.repeat_interleave(torch.arange(case["batch"]), torch.tensor(rows)).to(device)
        s["row_index"] = torch.cat([torch.arange(n) for n in rows]).to(device)
        s["rows"] = torch.tensor(rows, device=device)
    if own:
        _handle(s, case)
    return s


# ── the plain forms ─────────────────────────────────────────────────────────────────────────────────────────────────
def _turn(x, angles, interleaved):
    """float32 heads `x` [..., dim] rotated by `angles` [..., pairs, (cosine, sine)]."""
    pairs = angles.shape[-2]
    c, n = angles[..., 0], angles[..., 1]
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _normed(x, weight):
    """Heads in float32, normed where there is a weight; the sum of squares in 64 bits."""
    if weight is None:
        return x.float()
    r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()
    return x.float() * r * weight.float()


def _codes(x, case):
    """Affine codes (packed words), scales and biases of float32 rows [..., dim].  The end of a group's range that is further from 0
    is a whole number of steps from 0 and kept as the bias; codes are the nearest to the scale and bias as the cache keeps them."""
    bits, group, dtype = case["bits"], case["group"], DTYPES[case["dtype"]]
    bins = float((1 << bits) - 1)
    x = x.unflatten(-1, (-1, group))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    wide = low.abs() > high.abs()
    span = high - low
    step = (span / bins).clamp(min=1e-7)
    edge = torch.where(wide, low, high)
    steps = torch.round(torch.where(span > 1e-7 * bins, edge * bins / span, edge / 1e-7).abs())
    none = steps == 0
    scale = torch.where(none, step, edge.abs() / steps)
    scale = torch.where(wide, scale, -scale).to(dtype)
    bias = torch.where(none, torch.zeros_like(edge), edge).to(dtype)
    codes = torch.round((x - bias.float()) / scale.float()).clamp(0, bins).to(torch.int32).flatten(-2)
    codes = codes.unflatten(-1, (-1, 32 // bits)) << torch.arange(0, 32, bits, dtype=torch.int32, device=x.device)
    return codes.sum(-1, dtype=torch.int32), scale.squeeze(-1), bias.squeeze(-1)


def _values(p, case, at=...):
    """The values that rows `at` of the pages stand for, in float32."""
    bits = case["bits"]
    words = p["codes"][at]
    codes = (words.unsqueeze(-1) >> torch.arange(0, 32, bits, dtype=torch.int32, device=words.device)) & ((1 << bits) - 1)
    codes = codes.flatten(-2).unflatten(-1, (-1, case["group"])).float()
    return (codes * p["scales"][at].float().unsqueeze(-1) + p["biases"][at].float().unsqueeze(-1)).flatten(-2)


def _plain_rope(s, case):
    position = s["offset"][:, None].long() + torch.arange(case["length"], device=s["offset"].device)
    angles = s["table"][position][:, None]
    turned = lambda name, weight: _turn(_normed(s[name], weight), angles, case["interleaved"]).to(s[name].dtype)
    if case["op"] == "rope":
        return turned("q", None)
    return turned("q", s["q_weight"]), turned("k", s["k_weight"])


def _plain_append(s, case):
    page, dtype = case["page"], s["k"].dtype
    real = s["positions"] >= 0
    position = s["positions"].clamp(min=0).long()
    angles = s["table"][position][:, None]
    spare = s["keys"]["codes"].shape[0] - 1
    at = torch.where(real, s["page_table"][s["sequences"].long(), position // page], spare).long()
    rows = (at, slice(None), position % page)
    for p, x in ((s["keys"], _turn(_normed(s["k"], s["k_weight"]), angles, case["interleaved"])), (s["values"], s["v"].float())):
        codes, scales, biases = _codes(x, case)
        p["codes"][rows], p["scales"][rows], p["biases"][rows] = codes, scales, biases
    out = {}
    if s["q"] is not None:
        out["q"] = _turn(_normed(s["q"], s["q_weight"]), angles, case["interleaved"]).to(dtype)
    for name in ("keys", "values"):
        out[name] = torch.where(real[:, None, None], _values(s[name], case, rows), 0.0).to(dtype)
    return out


def _plain_attention(s, case):
    batch, heads, key_heads, dim = case["batch"], case["heads"], case["key_heads"], case["dim"]
    rep, most = heads // key_heads, max(_lengths(case)[0])
    keys, values = (_values(s[name], case, s["page_table"].long()).transpose(1, 2).reshape(batch, key_heads, -1, dim) for name in ("keys", "values"))
    spread = s["q"].new_zeros((batch, most, heads, dim), dtype=torch.float32)
    spread[s["row_sequence"], s["row_index"]] = s["q"].float()
    spread = spread.reshape(batch, most, key_heads, rep, dim).permute(0, 2, 3, 1, 4).reshape(batch, key_heads, rep * most, dim)
    scores = (spread @ keys.transpose(-1, -2)).mul_(s["scale"]).reshape(batch, key_heads, rep, most, -1)
    key = torch.arange(scores.shape[-1], device=scores.device)
    last = s["lengths"].long()[:, None] - s["rows"][:, None] + torch.arange(most, device=scores.device)  # the last key a row sees
    seen = (key <= last[..., None]) & (key < s["lengths"].long()[:, None, None])
    if case["window"]:
        seen &= key > last[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].float().reshape(1, key_heads, rep, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isfinite(top), top, 0.0)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    out = weights.reshape(batch, key_heads, rep * most, -1) @ values
    out = torch.where(total > 0, out.reshape(batch, key_heads, rep, most, dim) / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    return out[s["row_sequence"], s["row_index"]].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"rope": _plain_rope, "norm": _plain_rope, "append": _plain_append, "attention": _plain_attention}[case["op"]](s, case)
    import nuvec_amd as nv
    if case["op"] == "rope":
        return nv.rope(s["q"], s["rotation"], s["offset"])
    if case["op"] == "norm":
        return nv.head_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rotation"], s["offset"], EPS)
    if case["op"] == "append":
        q = nv.append_paged(s["cache"], s["k"], s["v"], s["page_table"], s["positions"], s["sequences"], s["rotation"],
                            k_weight=s["k_weight"], q=s["q"], q_weight=s["q_weight"], eps=EPS)
        keys, values = nv.read_paged(s["cache"], s["page_table"], s["positions"], s["sequences"])
        return {"keys": keys, "values": values} if q is None else {"q": q, "keys": keys, "values": values}
    return nv.paged_attention(s["q"], s["cache"], s["page_table"], s["lengths"], s["scale"], query_starts=s["starts"],
                              max_queries=case["queries"], sinks=s["sinks"], window=case["window"])


# ── the floor and the definition ────────────────────────────────────────────────────────────────────────────────────
def work(case):
    size, dim = DTYPE_BYTES[case["dtype"]], case["dim"]
    if case["op"] in ("rope", "norm"):
        rows = case["batch"] * case["length"]
        values = rows * (case["heads"] + case.get("key_heads", 0)) * dim
        return {"bytes": 2 * size * values + 4 * rows * case["rotary"], "flops": (7 if case["op"] == "norm" else 3) * values}
    row = dim * case["bits"] // 8 + 2 * size * dim // case["group"]  # bytes of a row of the cache
    if case["op"] == "append":
        tokens, kv = case["tokens"], case["key_heads"]
        queries = case["heads"] if case["queries"] else 0
        # read and written: the queries; the keys and values, their codes, and the values that the codes stand for
        moved = 2 * size * queries * dim + 2 * kv * (2 * size * dim + 2 * row) + 4 * case["rotary"]
        return {"bytes": tokens * moved, "flops": tokens * dim * (3 * queries + 20 * kv)}
    rows, positions = _lengths(case)
    read = seen = 0
    for n, length in zip(rows, positions):
        first = max(0, length - n - case["window"] + 1) if case["window"] else 0
        read += max(0, length - first)
        for i in range(n):
            last = length - n + i
            seen += max(0, last + 1 - (max(0, last - case["window"] + 1) if case["window"] else 0))
    return {"bytes": 2 * read * case["key_heads"] * row + 2 * size * sum(rows) * case["heads"] * dim, "flops": 4 * seen * case["heads"] * dim}


def _exact_turn(x, table, interleaved):
    y = x.clone()
    half = table.shape[-2]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    c, n = table[..., 0], table[..., 1]
    y[..., first] = x[..., first] * c - x[..., second] * n
    y[..., second] = x[..., first] * n + x[..., second] * c
    return y


def _exact_norm(x, weight):
    x = x.double()
    return x if weight is None else x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()


def _exact_stored(x, case):
    """What the cache stands for: of each group the end further from 0 as the bias, a step that divides it into a whole number nearest
    to what the range asks for, both kept in the element type, and every value's nearest multiple of that step from that bias."""
    bins, dtype = 2 ** case["bits"] - 1, DTYPES[case["dtype"]]
    kept = lambda t: t.to(dtype).double()
    parts = []
    for part in x.split(case["group"], -1):
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        falling = high.abs() >= low.abs()  # codes count down from the upper end
        edge = torch.where(falling, high, low)
        count = torch.where(high - low > 1e-7 * bins, edge.abs() * bins / (high - low), edge.abs() * 1e7).round()
        whole = edge.abs() / count.clamp_min(1)
        size = torch.where(count > 0, whole, ((high - low) / bins).clamp_min(1e-7))
        scale, bias = kept(torch.where(falling, -size, size)), kept(torch.where(count > 0, edge, 0.0))
        parts.append(((part - bias) / scale).round().clamp(0, bins) * scale + bias)
    return torch.cat(parts, -1)


def _exact_rows(p, case, pages, length):
    """A sequence's rows [key heads, length, dim] in 64 bits."""
    per, codes = 32 // case["bits"], p["codes"][pages].long() & 0xFFFFFFFF
    codes = torch.stack([(codes >> (case["bits"] * i)) % (1 << case["bits"]) for i in range(per)], -1).flatten(-2).double()
    wide = lambda t: t[pages].double().repeat_interleave(case["group"], -1)
    rows = codes * wide(p["scales"]) + wide(p["biases"])
    return rows.transpose(0, 1).flatten(1, 2)[:, :length]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rope", "norm"):
        at = torch.stack([torch.arange(case["length"], device="cuda") + int(o) for o in s["offset"].tolist()])
        table = s["table"].double()[at].unsqueeze(1)
        if case["op"] == "rope":
            return _exact_turn(s["q"].double(), table, case["interleaved"])
        return tuple(_exact_turn(_exact_norm(s[n], s[n + "_weight"]), table, case["interleaved"]) for n in ("q", "k"))
    if case["op"] == "append":
        padding = (s["positions"] < 0)[:, None, None]
        table = s["table"].double()[s["positions"].clamp(min=0).long()].unsqueeze(1)
        keys = _exact_stored(_exact_turn(_exact_norm(s["k"], s["k_weight"]), table, case["interleaved"]), case)
        out = {"keys": keys.masked_fill(padding, 0), "values": _exact_stored(s["v"].double(), case).masked_fill(padding, 0)}
        if s["q"] is not None:
            out["q"] = _exact_turn(_exact_norm(s["q"], s["q_weight"]), table, case["interleaved"])
        return out
    rows, positions = _lengths(case)
    rep, out, at = case["heads"] // case["key_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, length) in enumerate(zip(rows, positions)):
        if length > 0:
            pages = s["page_table"][b, :-(-length // case["page"])].long()
            keys, values = _exact_rows(s["keys"], case, pages, length), _exact_rows(s["values"], case, pages, length)
            behind = (length - n + torch.arange(n, device="cuda"))[:, None] - torch.arange(length, device="cuda")  # positions that a key lies behind a row
            hidden = (behind < 0) | (behind >= case["window"]) if case["window"] else behind < 0
            for h in range(case["heads"]):
                score = (s["q"][at:at + n, h].double() @ keys[h // rep].T * case["dim"] ** -0.5).masked_fill(hidden, -math.inf)
                if s["sinks"] is not None:
                    score = torch.cat([score, s["sinks"][h].double().expand(n, 1)], -1)
                weight = torch.softmax(score, -1).nan_to_num(0.0)[:, :length]  # (a row that sees nothing: zeros)
                out[at:at + n, h] = weight @ values[h // rep]
        at += n
    return out
