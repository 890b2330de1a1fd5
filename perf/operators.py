"""Measured cases of the decoder-side operators: RMS norm with residual and int8 output, the paged
key-value cache's append, and attention over that cache for prompts and for single tokens.

Each case runs either in its plain form (elementary torch operations in 32 bits) or, with ``own``
set, through the package's public entry points.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5
_ATTN_SCALE = 1.0 / 32.0  # int8 step of an attention output: values are of order 1, |v| < 4


def listed():
    return [
        # one token through a decoder layer's norm: latency
        {"name": "rmsnorm one token", "op": "rmsnorm", "rows": 1, "d": 4096, "x": "f16", "residual": "f16",
         "out": "same"},
        # the encoder block's shape (32 x 384 tokens of 768), residual stream in f32, input of an INT8 projection
        {"name": "rmsnorm block int8", "op": "rmsnorm", "rows": 12288, "d": 768, "x": "f32", "residual": "f32",
         "out": "int8 row"},
        # a large prompt batch of a wide model
        {"name": "rmsnorm wide bf16", "op": "rmsnorm", "rows": 16384, "d": 8192, "x": "bf16", "residual": "bf16",
         "out": "same"},
        # one new token for each of 64 sequences
        {"name": "append tokens", "op": "append", "type": "f16", "batch": 64, "heads": 8, "d": 128, "page": 64,
         "longest": 2048, "new": 1},
        # prompts of a ragged batch
        {"name": "append prompts", "op": "append", "type": "bf16", "batch": 16, "heads": 8, "d": 128, "page": 16,
         "longest": 4096, "new": 4096},
        # a short prompt, the encoder block's heads
        {"name": "prefill short", "op": "prefill", "type": "f16", "batch": 1, "heads": 12, "group": 1, "d": 64,
         "page": 16, "longest": 100, "new": 100, "window": 0, "sinks": 0, "out": "same"},
        # a ragged batch of prompts, grouped heads
        {"name": "prefill ragged", "op": "prefill", "type": "bf16", "batch": 8, "heads": 8, "group": 4, "d": 128,
         "page": 64, "longest": 2048, "new": 2048, "window": 0, "sinks": 0, "out": "same"},
        # one long prompt
        {"name": "prefill long", "op": "prefill", "type": "f16", "batch": 1, "heads": 8, "group": 4, "d": 128,
         "page": 64, "longest": 8192, "new": 8192, "window": 0, "sinks": 0, "out": "same"},
        # one long prompt under a sliding window with four sinks
        {"name": "prefill window", "op": "prefill", "type": "f16", "batch": 1, "heads": 4, "group": 4, "d": 64,
         "page": 32, "longest": 8192, "new": 8192, "window": 1024, "sinks": 4, "out": "same"},
        # the next token of one short sequence: latency
        {"name": "decode short", "op": "decode", "type": "f16", "batch": 1, "heads": 12, "group": 1, "d": 64,
         "page": 16, "longest": 200, "window": 0, "sinks": 0, "out": "same"},
        # the next token of one very long sequence: few rows, split over the cache
        {"name": "decode long", "op": "decode", "type": "bf16", "batch": 1, "heads": 8, "group": 4, "d": 128,
         "page": 64, "longest": 131072, "window": 0, "sinks": 0, "out": "same"},
        # the next tokens of a ragged batch
        {"name": "decode batch", "op": "decode", "type": "f16", "batch": 64, "heads": 8, "group": 4, "d": 128,
         "page": 16, "longest": 8192, "window": 0, "sinks": 0, "out": "same"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rmsnorm", "append", "prefill", "prefill", "decode", "decode"])
    if op == "rmsnorm":
        d = _log(rng, 64, 16384)
        if rng.random() < 0.75:
            d = max(64, d // 8 * 8)
        x = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "rows": _log(rng, 1, min(16384, 134217728 // (2 * d))), "d": d, "x": x,
                "residual": rng.choice([x, "f32", "none"]), "out": rng.choice(["same", "int8", "int8 row"])}
    page = rng.choice([8, 16, 32, 64, 128, 256])
    kind = rng.choice(["f16", "bf16"])
    d = rng.choice([64, 128])
    if op == "append":
        longest = _log(rng, 1, 4096)
        return {"op": op, "type": kind, "batch": _log(rng, 1, 16), "heads": _log(rng, 1, 16) if d == 64 else _log(rng, 1, 8),
                "d": d, "page": page, "longest": longest, "new": longest if rng.random() < 0.5 else 1}
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    sinks = rng.choice([0, 1, 4, 5, 100])
    case = {"op": op, "type": kind, "batch": 1, "heads": 1, "group": group, "d": d, "page": page, "longest": 0,
            "window": 0, "sinks": 0, "out": rng.choice(["same", "same", "same", "int8"])}
    if op == "prefill":
        # batch * heads * group * longest^2 stays below the long prompt's
        longest = _log(rng, 2, 8192)
        room = 32 * 8192 * 8192 // (longest * longest)
        case["heads"] = _log(rng, 1, max(1, min(8, room // group)))
        case["batch"] = _log(rng, 1, max(1, min(16, room // (group * case["heads"]))))
        case["longest"] = longest
        case["new"] = longest if rng.random() < 0.6 else _log(rng, 1, longest)
    else:
        longest = _log(rng, 2, 131072)
        room = 131072 * 8 * 128 // (longest * d)
        case["heads"] = _log(rng, 1, max(1, min(16, room)))
        case["batch"] = _log(rng, 1, max(1, min(256, room // case["heads"])))
        case["longest"] = longest
    if rng.random() < 0.5:
        case["window"] = _log(rng, 1, 2 * case["longest"])
        case["sinks"] = sinks
    return case


def _lengths(case):
    """Tokens in the cache (the new ones among them) and new tokens of each sequence: the first is
    the longest, the others are spread below it."""
    longest = case["longest"]
    total = [longest] + [max(1, int(longest * ((0.5 + 0.6180339887 * b) % 1.0))) for b in range(1, case["batch"])]
    return total, [min(n, case.get("new", 1)) for n in total]


def _visible(case, total, new):
    """(keys that some query sees, visible (query, key) pairs) of one sequence."""
    window, sinks = case["window"], case["sinks"]
    first = total - new  # position of the first query
    if window == 0:
        return total, new * first + new * (new + 1) // 2
    low = max(0, first - window + 1)
    keys = total - low + min(sinks, low)
    pairs = 0
    # queries at p < window see p + 1 keys; the later ones `window` keys and the sinks before them
    early = max(0, min(total, window) - first)
    pairs += early * first + early * (early + 1) // 2
    p0 = first + early  # the first query whose window does not reach the start
    late = total - p0
    if late > 0:
        pairs += late * window
        # sinks visible beside the window of the query at p: min(sinks, p - window + 1)
        grow = max(0, min(total, window - 1 + sinks) - p0)
        pairs += grow * (p0 - window + 1) + grow * (grow - 1) // 2 + (late - grow) * sinks
    return keys, pairs


def work(case):
    if case["op"] == "rmsnorm":
        size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
        n = case["rows"] * case["d"]
        out = {"same": size[case["x"]], "int8": 1, "int8 row": 1}[case["out"]]
        b = n * (size[case["x"]] + 2 * size[case["residual"]] + out) + 4 * case["d"]
        return {"bytes": b + (4 * case["rows"] if case["out"] == "int8 row" else 0), "flops": 5 * n}
    total, new = _lengths(case)
    row = case["heads"] * case["d"] * 2  # bytes of one token's keys
    if case["op"] == "append":
        return {"bytes": 4 * row * sum(new), "flops": 0}
    seen = [_visible(case, t, n) for t, n in zip(total, new)]
    q = sum(new) * row * case["group"]
    b = 2 * row * sum(k for k, _ in seen) + q + (q if case["out"] == "same" else q // 2)
    return {"bytes": b, "flops": 4 * case["d"] * case["heads"] * case["group"] * sum(p for _, p in seen)}


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["op"] == "rmsnorm":
        rows, d, t = case["rows"], case["d"], _TYPES[case["x"]]
        s = {"x": normal(rows, d, dtype=t), "gamma": 1.0 + 0.1 * normal(d), "s_out": 4.0 / 127.0}
        if case["residual"] != "none":
            s["residual"] = normal(rows, d, dtype=_TYPES[case["residual"]]) * 2.0
            s["sum"] = torch.empty_like(s["residual"])
        if case["out"] == "same":
            s["out"] = torch.empty_like(s["x"])
        else:
            s["q"] = torch.empty(rows, d, dtype=torch.int8, device=dev)
            s["values"] = torch.empty(rows, d, dtype=torch.float16, device=dev)
            if case["out"] == "int8 row":
                s["scales"] = torch.empty(rows, dtype=torch.float32, device=dev)
        return {"case": dict(case), **s}

    total, new = _lengths(case)
    t, batch, page, heads, d = _TYPES[case["type"]], case["batch"], case["page"], case["heads"], case["d"]
    most = -(-max(total) // page)
    pages = sum(-(-n // page) for n in total)
    count = pages + 3
    order = torch.randperm(count, generator=g, device=dev).to(torch.int32)
    # each sequence's pages anywhere in the cache; table entries behind its last page hold -1
    used = torch.tensor([-(-n // page) for n in total], device=dev)
    column = torch.arange(most, device=dev)
    start = torch.cumsum(used, 0) - used
    table = torch.where(column[None] < used[:, None], order[(start[:, None] + column[None]).clamp(max=count - 1)], -1)
    lens = torch.tensor(total, dtype=torch.int32, device=dev)
    k = normal(count, page, heads, d, dtype=t)
    v = normal(count, page, heads, d, dtype=t)
    s = {"case": dict(case), "k": k, "v": v, "table": table.to(torch.int32), "lens": lens, "total": total, "new": new}
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
    tokens = offsets[-1]
    if case["op"] == "append":
        s["new_k"] = normal(tokens, heads, d, dtype=t)
        s["new_v"] = normal(tokens, heads, d, dtype=t)
    else:
        # slots that no token has been written to hold what was there before: here NaN
        last = torch.tensor([n - 1 for n in total], device=dev)
        tail = s["table"].long()[torch.arange(batch, device=dev), last // page]
        slot = torch.arange(page, device=dev)
        behind = slot[None] > (last % page)[:, None]
        for c in (k, v):
            c[tail] = torch.where(behind[:, :, None, None], float("nan"), c[tail])
        s["q"] = normal(tokens, heads * case["group"], d, dtype=t) * 2.0  # scores of deviation 2
        if case["out"] == "same":
            s["out"] = torch.empty_like(s["q"])
        else:
            s["q8"] = torch.empty(s["q"].shape, dtype=torch.int8, device=dev)
            s["values"] = torch.empty(s["q"].shape, dtype=torch.float16, device=dev)
    if own:
        from lightship_b200.kv_cache import PagedKVCache
        s["cache"] = PagedKVCache(k, v, s["table"], lens)
    return s


def _plain_rmsnorm(s):
    c = s["case"]
    h = s["x"].float()
    outs = []
    if c["residual"] != "none":
        h = h + s["residual"].float()
        outs.append(h.to(s["residual"].dtype))
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS) * s["gamma"]
    if c["out"] == "same":
        return outs + [y.to(s["x"].dtype)]
    scale = torch.full((c["rows"],), s["s_out"], device=y.device)
    if c["out"] == "int8 row":
        top = y.abs().amax(1)
        scale = torch.where(top > 0, top / 127.0, torch.ones_like(top))
        outs.append(scale)
    t = y / scale[:, None]
    q = (torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-128, 127)
    return outs + [(q * scale[:, None]).half()]


def _positions(s):
    """[batch, most new] positions of the new tokens, their rows in the packed batch, and which exist."""
    new = torch.diff(s["offsets"])
    i = torch.arange(max(s["new"]), device=new.device)
    there = i[None] < new[:, None]
    return (s["lens"] - new)[:, None] + i[None], s["offsets"][:-1, None] + i[None], there


def _plain_append(s):
    page = s["case"]["page"]
    pos, row, there = _positions(s)
    pos = torch.where(there, pos, 0).long()
    at = torch.gather(s["table"].long(), 1, pos // page)[there]
    slot = (pos % page)[there]
    s["k"][at, slot] = s["new_k"][row[there].long()]
    s["v"][at, slot] = s["new_v"][row[there].long()]
    return [s["k"], s["v"]]


def _plain_attention(s):
    c = s["case"]
    page, heads, group, d = c["page"], c["heads"], c["group"], c["d"]
    batch, longest = c["batch"], max(s["total"])
    j = torch.arange(longest, device=s["q"].device)
    held = j[None] < s["lens"][:, None]
    at = torch.where(held, s["table"].long()[:, j // page], 0)
    slot = (j % page)[None].expand(batch, -1)
    live = held[:, :, None, None]
    k = torch.where(live, s["k"][at, slot], 0).float().permute(0, 2, 1, 3)  # [batch, heads, longest, d]
    v = torch.where(live, s["v"][at, slot], 0).float().permute(0, 2, 1, 3)
    pos, row, there = _positions(s)
    n = pos.shape[1]
    q = s["q"][torch.where(there, row, 0).long()].float()  # [batch, n, heads * group, d]
    q = q.view(batch, n, heads, group, d).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * n, d)
    mask = (j[None, None] <= pos[:, :, None]) & held[:, None]
    if c["window"] > 0:
        mask &= (j[None, None] > pos[:, :, None] - c["window"]) | (j < c["sinks"])[None, None]
    scores = (q @ k.transpose(2, 3)).view(batch, heads, group, n, longest)
    scores.mul_(1.0 / math.sqrt(d)).masked_fill_(~mask[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weight = scores.sub_(top).exp_()
    norm = weight.sum(-1, keepdim=True)
    o = weight.view(batch, heads, group * n, longest) @ v
    o = o.view(batch, heads, group, n, d) / torch.where(norm > 0, norm, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, n, heads * group, d)[there]
    if c["out"] == "same":
        return [o.to(s["q"].dtype)]
    t = o / _ATTN_SCALE
    q8 = (torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-128, 127)
    return [(q8 * _ATTN_SCALE).half()]


def run(state):
    c = state["case"]
    if not own:
        return {"rmsnorm": _plain_rmsnorm, "append": _plain_append}.get(c["op"], _plain_attention)(state)
    if c["op"] == "rmsnorm":
        from lightship_b200 import ops
        ops.rmsnorm(state["x"], state["gamma"], eps=_EPS, residual=state.get("residual"), sum_out=state.get("sum"),
                    out=state.get("out"), out_i8=state.get("q"), s_out=state["s_out"] if c["out"] == "int8" else 0.0,
                    row_scales=state.get("scales"))
        outs = [state["sum"]] if "sum" in state else []
        if c["out"] == "same":
            return outs + [state["out"]]
        if c["out"] == "int8 row":
            outs.append(state["scales"])
            return outs + [torch.mul(state["q"], state["scales"][:, None], out=state["values"])]
        return outs + [torch.mul(state["q"], state["s_out"], out=state["values"])]
    cache = state["cache"]
    if c["op"] == "append":
        cache.append(state["new_k"], state["new_v"], state["offsets"])
        return [state["k"], state["v"]]
    more = {"alpha": 1.0 / math.sqrt(c["d"]), "window": c["window"], "sinks": c["sinks"]}
    more.update({"out": state["out"]} if c["out"] == "same" else {"out_i8": state["q8"], "s_out": _ATTN_SCALE})
    if c["op"] == "prefill":
        cache.prefill(state["q"], state["offsets"], **more)
    else:
        cache.decode(state["q"], **more)
    if c["out"] == "same":
        return [state["out"]]
    return [torch.mul(state["q8"], _ATTN_SCALE, out=state["values"])]


def _round_half_away(t):
    down = torch.floor(t.abs())
    return torch.sign(t) * torch.where(t.abs() - down >= 0.5, down + 1, down)


def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    if case["op"] == "rmsnorm":
        outs, h = [], s["x"].double()
        if case["residual"] != "none":
            h = h + s["residual"].double()
            outs.append(h)
        y = h / torch.sqrt((h ** 2).sum(-1, keepdim=True) / case["d"] + _EPS) * s["gamma"].double()
        if case["out"] == "same":
            return outs + [y]
        scale = torch.full_like(y[:, :1], s["s_out"])
        if case["out"] == "int8 row":
            scale = y.abs().max(1, keepdim=True).values / 127
            scale[scale == 0] = 1.0
            outs.append(scale[:, 0])
        return outs + [_round_half_away(y / scale).clamp(-128, 127) * scale]
    table, offsets = s["table"].long().cpu(), s["offsets"].tolist()
    total, new, page = s["total"], s["new"], case["page"]
    if case["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        for b in range(case["batch"]):
            pos = torch.arange(total[b] - new[b], total[b])
            at, slot = table[b][pos // page].to(k.device), (pos % page).to(k.device)
            k[at, slot] = s["new_k"][offsets[b]:offsets[b + 1]].double()
            v[at, slot] = s["new_v"][offsets[b]:offsets[b + 1]].double()
        return [k, v]
    group, d, window = case["group"], case["d"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(case["batch"]):
        n, used = total[b], -(-total[b] // page)
        ids = table[b][:used].to(out.device)
        for h in range(case["heads"]):
            k = s["k"][ids, :, h].reshape(-1, d)[:n].double()
            v = s["v"][ids, :, h].reshape(-1, d)[:n].double()
            for i in range(0, new[b], 2048):
                rows = slice(offsets[b] + i, offsets[b] + min(new[b], i + 2048))
                p = torch.arange(n - new[b] + i, n - new[b] + min(new[b], i + 2048), device=out.device)
                j = torch.arange(n, device=out.device)
                hidden = j[None] > p[:, None]
                if window > 0:
                    hidden |= (j[None] <= p[:, None] - window) & (j[None] >= case["sinks"])
                for a in range(group):
                    z = s["q"][rows, h * group + a].double() @ k.T / d ** 0.5
                    z[hidden] = float("-inf")
                    out[rows, h * group + a] = torch.softmax(z, -1) @ v
    if case["out"] == "same":
        return [out]
    return [_round_half_away(out / _ATTN_SCALE).clamp(-128, 127) * _ATTN_SCALE]
