"""More operators of a decoder block that serves many requests, as cases that can be timed and compared.

A case is a dict of plain values; its `op` names the operator:

  prompt      attention over whole prompts of several sequences, keys and values as the projections leave them (`prompt_attention`)
  adapters    low-rank adapters of many requests beside a shared projection (`apply_adapters`)
  select      the choice of experts: scores, a bias, groups, the best of them and their weights (`moe_select`)
  axes        rotary positions with an axis each for time, height and width, with or without the heads' norms (`rope`, `head_norm_rope`)

With `own` false `run` computes them in elementary torch operations, in 32 bits (the choice of experts and the sums of squares in 64: what
lies next to a border falls on one side of it); with `own` true it makes the package's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
DTYPE_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}
EPS = 1e-6

# The largest work of a drawn case, that of the largest listed ones: a prompt of 8192 tokens in 32 heads of 128, 4096 tokens beside a
# [14336, 4096] projection, the logits of 16384 tokens, two prompts of 2049 tokens in 40 heads.
MOST_SCORES = 32 * 8192 * 8192
MOST_PRODUCTS = 32 * 8192 * 8192 // 2 * 128
MOST_PROJECTED = 4096 * (4096 + 2 * 14336)
MOST_ADAPTED = 64 * 32 * (4096 + 14336)
MOST_LOGITS = 16384 * 256
MOST_VALUES = 2 * 2049 * 40 * 128


def listed():
    return [
        # Short prompts of seven requests that arrive together, one of a single token: the smallest call.
        {"name": "prompt_short", "op": "prompt", "dtype": "bfloat16", "heads": 32, "key_heads": 8, "dim": 128, "batch": 7, "rows": 61,
         "prefix": 0, "sinks": False, "window": 0},
        # One long prompt: two matrix products with a softmax between them.
        {"name": "prompt_long", "op": "prompt", "dtype": "bfloat16", "heads": 32, "key_heads": 8, "dim": 128, "batch": 1, "rows": 8192,
         "prefix": 0, "sinks": False, "window": 0},
        # Ragged chunks of several prompts, some with earlier keys in front of them, sinks and a sliding window, small heads.
        {"name": "prompt_ragged", "op": "prompt", "dtype": "float16", "heads": 20, "key_heads": 5, "dim": 64, "batch": 9, "rows": 1500,
         "prefix": 700, "sinks": True, "window": 1000},
        # The next tokens of 64 requests, each with an adapter of its own: every adapter's weights come from memory.
        {"name": "adapters_step", "op": "adapters", "dtype": "bfloat16", "rows": 64, "k": 4096, "n": 4096, "rank": 16, "adapters": 64,
         "runs": False},
        # Prompts of a few requests beside the widest projection.
        {"name": "adapters_prompt", "op": "adapters", "dtype": "bfloat16", "rows": 4096, "k": 4096, "n": 14336, "rank": 32, "adapters": 4,
         "runs": True},
        # Chunks and single tokens, sizes that are no whole tiles.
        {"name": "adapters_ragged", "op": "adapters", "dtype": "float16", "rows": 517, "k": 2880, "n": 2880, "rank": 12, "adapters": 9,
         "runs": True},
        # A decode step of eight requests: sigmoid scores with a bias, four of eight groups, eight of 256 experts.
        {"name": "select_step", "op": "select", "dtype": "float32", "rows": 8, "experts": 256, "k": 8, "scores": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "normalize": True, "scale": 2.5},
        # The tokens of a long prompt through the same router.
        {"name": "select_prompt", "op": "select", "dtype": "bfloat16", "rows": 16384, "experts": 256, "k": 8, "scores": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "normalize": True, "scale": 2.5},
        # Softmax scores of a number of experts that fills no wavefront, no groups, weights as they are.
        {"name": "select_ragged", "op": "select", "dtype": "float16", "rows": 1333, "experts": 60, "k": 4, "scores": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "normalize": False, "scale": 1.0},
        # The next tokens of eight requests, behind images.
        {"name": "axes_step", "op": "axes", "dtype": "bfloat16", "norm": True, "batch": 8, "heads": 32, "key_heads": 8, "length": 1,
         "dim": 128, "rotary": 128, "time": 24, "height": 20, "width": 20, "dealt": True, "interleaved": False, "table": 32768},
        # Two prompts of text and images, queries and keys normed and rotated.
        {"name": "axes_prompt", "op": "axes", "dtype": "bfloat16", "norm": True, "batch": 2, "heads": 32, "key_heads": 8, "length": 2049,
         "dim": 128, "rotary": 128, "time": 24, "height": 20, "width": 20, "dealt": True, "interleaved": False, "table": 32768},
        # The patches of images: height and width alone, neighbouring values paired, a head size that is no power of two.
        {"name": "axes_image", "op": "axes", "dtype": "float16", "norm": False, "batch": 3, "heads": 16, "key_heads": 0, "length": 1025,
         "dim": 80, "rotary": 80, "time": 0, "height": 20, "width": 20, "dealt": False, "interleaved": True, "table": 4096},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: its operator and types by how often they are met, its sizes over the whole range."""
    most = {}
    for case in listed():
        for what, amount in work(case).items():
            most[case["op"], what] = max(amount, most.get((case["op"], what), 0))
    while True:
        case = _draw(rng)
        if all(amount <= most[case["op"], what] for what, amount in work(case).items()):
            return case


def _draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "adapters", "adapters", "adapters", "select", "select", "axes"])
    c = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "bfloat16", "float16", "float16", "float32"])}
    if op == "prompt":
        key_heads = rng.choice([1, 2, 4, 5, 8, 8])
        heads = key_heads * rng.choice([1, 2, 3, 4, 4, 8])
        batch, dim = _log(rng, 1, 16), rng.choice([64, 80, 96, 128, 128, 128, 256])
        rows = _log(rng, 1, 8192 // batch)
        prefix = rng.choice([0, 0, _log(rng, 1, 4096)])
        while batch * heads * rows * (rows + prefix) > MOST_SCORES or batch * heads * rows * (rows + 2 * prefix) // 2 * dim > MOST_PRODUCTS:
            rows, prefix = rows // 2 + 1, prefix // 2
        c.update(heads=heads, key_heads=key_heads, dim=dim, batch=batch, rows=rows, prefix=prefix, sinks=rng.random() < 0.3,
                 window=rng.choice([0, 0, 0, _log(rng, 16, 2048)]))
    elif op == "adapters":
        count, rank = _log(rng, 1, 64), rng.choice([4, 8, 8, 12, 16, 16, 16, 32, 32, 64, 128])
        k, n = _log(rng, 256, 14336), _log(rng, 256, 14336)
        k, n = (k, n) if rng.random() < 0.15 else (k // 32 * 32, n // 32 * 32)
        while count * rank * (k + n) > MOST_ADAPTED:
            count = (count + 1) // 2 if count > 1 else 1
            if count == 1:
                rank = min(rank, 64)
                break
        rows = _log(rng, 1, min(4096, MOST_PROJECTED // (k + 2 * n) * 2 // DTYPE_BYTES[c["dtype"]]))
        c.update(rows=rows, k=k, n=n, rank=rank, adapters=count, runs=rows > 16 and rng.random() < 0.7)
    elif op == "select":
        experts, k, groups = rng.choice([(8, 2, 1), (16, 1, 1), (32, 4, 1), (60, 4, 1), (64, 6, 1), (64, 8, 8), (128, 8, 1), (160, 6, 8),
                                         (256, 8, 8), (256, 8, 1), (384, 8, 1), (512, 10, 1)])
        scores = rng.choice(["softmax", "sigmoid"])
        c.update(rows=_log(rng, 1, MOST_LOGITS // max(256, experts)), experts=experts, k=k, scores=scores, bias=rng.random() < 0.6, groups=groups,
                 top_groups=1 if groups == 1 else rng.choice([3, 4]), normalize=rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 2.5]))
    else:
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        c.update(norm=rng.random() < 0.6, batch=_log(rng, 1, 32), heads=_log(rng, 1, 64), dim=dim, rotary=rng.choice([dim, dim, dim // 2]),
                 dealt=rng.random() < 0.5, interleaved=rng.random() < 0.3, table=rng.choice([8192, 32768]))
        c["key_heads"] = _log(rng, 1, 16) if c["norm"] else 0
        pairs = c["rotary"] // 2
        c["time"] = rng.choice([0, pairs // 4, pairs // 3 + 1])
        c["height"] = (pairs - c["time"]) // 2
        c["width"] = pairs - c["time"] - c["height"]
        most = MOST_VALUES * 2 // DTYPE_BYTES[c["dtype"]] // (c["batch"] * (c["heads"] + c["key_heads"]) * dim)
        c["length"] = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, min(4096, most)))
    return c


# ── inputs ──────────────────────────────────────────────────────────────────────────────────────────────────────────
def _sequences(case):
    """(rows, keys) of each sequence: whole prompts and shorter ones, single tokens, those behind a prefix; in larger batches one has no
    rows and one more rows than keys."""
    out = []
    for b in range(case["batch"]):
        n = (case["rows"], max(1, case["rows"] // 2), 1, max(1, case["rows"] // 3 + 1))[b % 4]
        keys = n + (case["prefix"], case["prefix"] // 3, case["prefix"])[b % 3]
        if b == 5:
            n = 0
        elif b == 7:
            n, keys = 3, 2
        out.append((n, keys))
    return out


def _axis_of(case):
    """The axis (0 time, 1 height, 2 width) of each pair: in consecutive runs, or dealt out in turn to the axes that have pairs left."""
    left = [case["time"], case["height"], case["width"]]
    if not case["dealt"]:
        return [a for a in range(3) for _ in range(left[a])]
    axes = []
    while len(axes) < case["rotary"] // 2:
        for a in range(3):
            if left[a] > 0:
                axes.append(a)
                left[a] -= 1
    return axes


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=device)
    whole = lambda low, high, *shape: torch.randint(low, high, shape, generator=g, device=device, dtype=torch.int32)
    s = {"case": case}
    if case["op"] == "prompt":
        counts = _sequences(case)
        total = lambda i: [sum(c[i] for c in counts[:b]) for b in range(len(counts) + 1)]
        s["starts"], s["key_starts"] = (torch.tensor(total(i), dtype=torch.int32, device=device) for i in (0, 1))
        spread = torch.exp(0.5 * normal(1, case["key_heads"], case["dim"]))  # (channels of keys differ in size)
        s["q"] = normal(total(0)[-1], case["heads"], case["dim"]).to(dtype)
        s["k"] = (normal(total(1)[-1], case["key_heads"], case["dim"]) * spread).to(dtype)
        s["v"] = normal(total(1)[-1], case["key_heads"], case["dim"]).to(dtype)
        s["sinks"] = normal(case["heads"]).to(dtype) if case["sinks"] else None
    elif case["op"] == "adapters":
        rows, k, n, rank, count = (case[name] for name in ("rows", "k", "n", "rank", "adapters"))
        s["x"], s["y"] = normal(rows, k).to(dtype), normal(rows, n).to(dtype)
        s["down"], s["up"] = (normal(count, rank, k) * k ** -0.5).to(dtype), (0.3 * normal(count, n, rank) * rank ** -0.5).to(dtype)
        s["scales"] = 0.5 + 1.5 * torch.rand(count, generator=g, device=device)
        if case["runs"]:  # consecutive rows are one request's: chunks of many lengths, single tokens; one request in eight has no adapter
            ends = whole(0, rows, max(1, min(3 * count, rows // 8)))
            run = (torch.arange(rows, device=device)[:, None] > ends).sum(-1)
            of_run = torch.rand(count, generator=g, device=device).argsort().to(torch.int32).repeat(4)
            of_run[7::8] = -1
            s["ids"] = of_run[run].contiguous()
        else:
            order = torch.rand(count, generator=g, device=device).argsort().to(torch.int32)
            s["ids"] = order.repeat(-(-rows // count))[:rows].contiguous()
            s["ids"][7::11] = -1
    elif case["op"] == "select":
        popular = 0.7 * normal(case["experts"])
        s["logits"] = (1.2 * normal(case["rows"], case["experts"]) + popular).to(dtype)
        s["bias"] = -0.1 * popular + 0.02 * normal(case["experts"]) if case["bias"] else None
    else:
        batch, length, dim = case["batch"], case["length"], case["dim"]
        inverse = 500000.0 ** (-torch.arange(case["rotary"] // 2, device=device, dtype=torch.float64) * 2 / case["rotary"])
        angle = torch.arange(case["table"], device=device, dtype=torch.float64)[:, None] * inverse
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        # Runs of 256 tokens: text, whose axes move together, and images of 16 x 16 patches at one time.
        at = torch.arange(length, device=device)
        image, patch, text = at // 256 % 2 == 1, at % 256, at // 512 * 272 + at % 256
        start = at // 512 * 272 + 256
        axes = torch.stack([torch.where(image, start, text), torch.where(image, start + patch // 16, text), torch.where(image, start + patch % 16, text)])
        s["positions"] = (axes[:, None] + whole(0, case["table"] - length - 16, batch)[None, :, None]).to(torch.int32).contiguous()
        for name, h in (("q", case["heads"]), ("k", case["key_heads"])):  # heads [batch, heads, length, dim] over tokens outermost
            if h > 0:
                s[name] = normal(batch, length, h, dim).to(dtype).transpose(1, 2)
                s[name + "_weight"] = (1 + 0.2 * normal(dim)).to(dtype) if case["norm"] else None
        s["axis"] = torch.tensor(_axis_of(case), device=device)
    if own:
        _handle(s, case)
    return s


def _handle(s, case):
    """What a program that uses the package keeps beside these tensors: its objects over them."""
    import nuvec_amd as nv
    if case["op"] == "adapters":
        s["adapters"] = nv.Adapters(s["down"], s["up"], s["scales"])
    elif case["op"] == "axes":
        axes = nv.rotary_axes((case["time"], case["height"], case["width"]), case["dealt"])
        s["rotation"] = nv.Rotation(s["table"], case["interleaved"], axes)


# ── the plain forms ─────────────────────────────────────────────────────────────────────────────────────────────────
def _plain_prompt(s, case):
    rep, out, at, key_at = case["heads"] // case["key_heads"], torch.zeros_like(s["q"]), 0, 0
    for n, length in _sequences(case):
        if n > 0 and length > 0:
            q = s["q"][at:at + n].float().transpose(0, 1)  # [heads, n, dim]
            k, v = (s[name][key_at:key_at + length].float().transpose(0, 1).repeat_interleave(rep, 0) for name in ("k", "v"))
            scores = torch.matmul(q, k.transpose(1, 2)).mul_(case["dim"] ** -0.5)
            last = (length - n + torch.arange(n, device=q.device))[:, None]
            key = torch.arange(length, device=q.device)
            hidden = key > last
            if case["window"]:
                hidden = hidden | (key <= last - case["window"])
            scores.masked_fill_(hidden, float("-inf"))
            top = scores.amax(-1, keepdim=True)
            if s["sinks"] is not None:
                sink = s["sinks"].float()[:, None, None]
                top = torch.maximum(top, sink)
            top = torch.where(torch.isfinite(top), top, 0.0)
            weights = scores.sub_(top).exp_()
            total = weights.sum(-1, keepdim=True)
            if s["sinks"] is not None:
                total = total + (sink - top).exp()
            y = torch.matmul(weights, v)
            out[at:at + n] = torch.where(total > 0, y / total, 0.0).transpose(0, 1).to(out.dtype)
        at, key_at = at + n, key_at + length
    return out


def _plain_adapters(s, case):
    x, y = s["x"].float(), s["y"].float()
    for a in range(case["adapters"]):
        low = (x @ s["down"][a].float().T) * s["scales"][a]
        y = torch.where((s["ids"] == a)[:, None], s["y"].float() + low @ s["up"][a].float().T, y)
    return y.to(s["y"].dtype)


def _plain_select(s, case):
    logits = s["logits"].double()
    if case["scores"] == "softmax":
        scores = (logits - logits.amax(-1, keepdim=True)).exp()
        scores = scores / scores.sum(-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + (-logits).exp())
    rank = scores + s["bias"].double() if s["bias"] is not None else scores
    groups = case["groups"]
    if groups > 1:
        grouped = rank.unflatten(-1, (groups, -1))
        best = grouped.sort(-1, descending=True).values[..., :2 if case["bias"] else 1].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices[..., :case["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, order, True)
        rank = torch.where(kept[..., None], grouped, float("-inf")).flatten(-2)
    chosen = rank.sort(dim=-1, descending=True, stable=True).indices[..., :case["k"]]
    weights = scores.gather(-1, chosen)
    if case["normalize"]:
        weights = weights / (weights.sum(-1, keepdim=True) + 1e-20)
    return chosen.to(torch.int32), (weights * case["scale"]).to(s["logits"].dtype)


def _plain_axes(s, case):
    # the angles of every token's pairs, each at its axis's position
    pair = torch.arange(case["rotary"] // 2, device=s["axis"].device)
    angles = s["table"][s["positions"][s["axis"]].permute(1, 2, 0).long(), pair][:, None]  # [batch, 1, length, pairs, 2]
    c, n = angles[..., 0], angles[..., 1]
    out = []
    for name in ("q", "k")[:1 if case["key_heads"] == 0 else 2]:
        x = s[name].float()
        if case["norm"]:
            x = x * torch.rsqrt(s[name].double().square().mean(-1, keepdim=True) + EPS).float() * s[name + "_weight"].float()
        turning, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
        if case["interleaved"]:
            a, b = turning[..., 0::2], turning[..., 1::2]
            turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
        else:
            a, b = turning.chunk(2, -1)
            turned = torch.cat([a * c - b * n, b * c + a * n], -1)
        out.append(torch.cat([turned, rest], -1).to(s[name].dtype))
    return out


def run(s):
    case = s["case"]
    if not own:
        return {"prompt": _plain_prompt, "adapters": _plain_adapters, "select": _plain_select, "axes": _plain_axes}[case["op"]](s, case)
    import nuvec_amd as nv
    if case["op"] == "prompt":
        return nv.prompt_attention(s["q"], s["k"], s["v"], case["dim"] ** -0.5, s["starts"], s["key_starts"], sinks=s["sinks"], window=case["window"])
    if case["op"] == "adapters":
        return nv.apply_adapters(s["y"], s["x"], s["adapters"], s["ids"])
    if case["op"] == "select":
        return nv.moe_select(s["logits"], case["k"], case["scores"], s["bias"], case["groups"], case["top_groups"], normalize=case["normalize"],
                             scale=case["scale"])
    if case["norm"]:
        return list(nv.head_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rotation"], s["positions"], EPS))
    return [nv.rope(s["q"], s["rotation"], s["positions"])]


# ── the floor and the definition ────────────────────────────────────────────────────────────────────────────────────
def work(case):
    size = DTYPE_BYTES[case["dtype"]]
    if case["op"] == "prompt":
        rows = keys = seen = 0
        window = case["window"]
        for n, length in _sequences(case):
            rows += n
            if n == 0:
                continue
            first = max(0, length - n - window + 1) if window else 0
            keys += length - first
            for last in range(length - n, length):  # of each row, the last key that it sees
                if last >= 0:
                    seen += last + 1 if window == 0 else min(last + 1, window)
        return {"bytes": 2 * size * case["dim"] * (rows * case["heads"] + keys * case["key_heads"]), "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["op"] == "adapters":
        rows, k, n, rank = (case[name] for name in ("rows", "k", "n", "rank"))
        used = min(case["adapters"], rows)
        return {"bytes": size * (rows * (k + 2 * n) + used * rank * (k + n)) + 4 * (rows + used), "flops": 2 * rows * rank * (k + n)}
    if case["op"] == "select":
        values = case["rows"] * case["experts"]
        return {"bytes": size * values + case["rows"] * case["k"] * (4 + size) + (4 * case["experts"] if case["bias"] else 0), "flops": 10 * values}
    tokens = case["batch"] * case["length"]
    values = tokens * (case["heads"] + case["key_heads"]) * case["dim"]
    return {"bytes": 2 * size * values + tokens * (12 + 4 * case["rotary"]), "flops": (7 if case["norm"] else 3) * values}


def _exact_prompt(s, case):
    rep, dim = case["heads"] // case["key_heads"], case["dim"]
    out, at, key_at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, 0
    for n, length in _sequences(case):
        if n > 0 and length > 0:
            behind = (length - n + torch.arange(n, device="cuda"))[:, None] - torch.arange(length, device="cuda")  # how far a key lies behind a row
            hidden = (behind < 0) | (behind >= case["window"]) if case["window"] else behind < 0
            for h in range(case["heads"]):
                keys, values = (s[name][key_at:key_at + length, h // rep].double() for name in ("k", "v"))
                score = (s["q"][at:at + n, h].double() @ keys.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                if s["sinks"] is not None:
                    score = torch.cat([score, s["sinks"][h].double().expand(n, 1)], -1)
                weight = torch.softmax(score, -1).nan_to_num(0.0)[:, :length]  # (a row that sees nothing: zeros)
                out[at:at + n, h] = weight @ values
        at, key_at = at + n, key_at + length
    return out


def _exact_adapters(s, case):
    out = s["y"].double()
    for a, rows in ((a, (s["ids"] == a).nonzero()[:, 0]) for a in s["ids"].unique().tolist() if a >= 0):
        product = s["up"][a].double() @ (s["down"][a].double() @ s["x"][rows].double().T)  # [n, rows]
        out[rows] += s["scales"][a].double() * product.T
    return out


def _exact_select(s, case):
    logits = s["logits"].double()
    scores = torch.softmax(logits, -1) if case["scores"] == "softmax" else torch.sigmoid(logits)
    rank = scores if s["bias"] is None else scores + s["bias"].double()
    rows, experts, each = case["rows"], case["experts"], case["experts"] // case["groups"]

    def first_best(t):  # the lowest index of each row's largest value
        return (t == t.amax(-1, keepdim=True)).to(torch.int8).argmax(-1, keepdim=True)

    if case["groups"] > 1:
        best = torch.zeros((rows, case["groups"]), dtype=torch.float64, device="cuda")
        for i in range(case["groups"]):
            part = rank[:, i * each:(i + 1) * each]
            best[:, i] = part.amax(-1)
            if case["bias"]:
                best[:, i] += part.scatter(-1, first_best(part), -math.inf).amax(-1)
        open_ = torch.full_like(rank, -math.inf)
        for _ in range(case["top_groups"]):
            group = first_best(best)
            best.scatter_(-1, group, -math.inf)
            member = torch.arange(experts, device="cuda") // each == group
            open_ = torch.where(member, rank, open_)
        rank = open_
    rank, chosen = rank.clone(), []
    for _ in range(case["k"]):
        chosen.append(first_best(rank))
        rank.scatter_(-1, chosen[-1], -math.inf)
    chosen = torch.cat(chosen, -1)
    weights = scores.gather(-1, chosen)
    if case["normalize"]:
        weights = weights / (weights.sum(-1, keepdim=True) + 1e-20)
    return chosen.to(torch.int32), case["scale"] * weights


def _exact_axes(s, case):
    out = []
    for name in ("q", "k")[:1 if case["key_heads"] == 0 else 2]:
        x = s[name].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * s[name + "_weight"].double()
        y = x.clone()
        for i, axis in enumerate(_axis_of(case)):
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["rotary"] // 2)
            turn = s["table"][s["positions"][axis].long(), i].double()[:, None]  # [batch, 1, length, 2]
            y[..., first] = x[..., first] * turn[..., 0] - x[..., second] * turn[..., 1]
            y[..., second] = x[..., first] * turn[..., 1] + x[..., second] * turn[..., 0]
        out.append(y)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "adapters": _exact_adapters, "select": _exact_select, "axes": _exact_axes}[case["op"]](s, case)
