"""Workloads of the attention side of a step, around the INT8 linears: rotary positions with several axes, block tables and
slot maps from request lengths, the 8-bit cache's writes, and attention over that cache.

Kinds of case ("op"):
- "rotary":    queries and keys of one projection rotated in one call;
- "plan":      slots, positions and block tables of a step's new tokens, from the requests' lengths on the GPU;
- "write":     a step's keys and values into the 8-bit cache, then the touched pages read back as the values they stand for;
- "attention": the step's queries over the cache.

Requests: "requests" of up to "past" cached and "new" new tokens; with "ragged" every request has lengths of its own (the first
one the longest), some of them no new token.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def rotary_case(tokens, q_heads, k_heads, head_dim, sections, dtype="bf16", ladder="axis", style="pairs", inverse=False, packed=True, far=0):
    s = (*sections, 0, 0)
    return {"op": "rotary", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim, "s0": s[0], "s1": s[1], "s2": s[2],
            "dtype": dtype, "ladder": ladder, "style": style, "inverse": inverse, "packed": packed, "far": far}


def plan_case(requests, past, new, block, ragged=True, tight=False):
    return {"op": "plan", "requests": requests, "past": past, "new": new, "block": block, "ragged": ragged, "tight": tight}


def write_case(requests, past, new, heads, head_dim, block, dtype="bf16", ragged=True, packed=True):
    return {"op": "write", "requests": requests, "past": past, "new": new, "heads": heads, "head_dim": head_dim, "block": block, "dtype": dtype,
            "ragged": ragged, "packed": packed}


def attention_case(requests, past, new, heads, group, head_dim, block, dtype="bf16", causal=True, window=0, ragged=True):
    return {"op": "attention", "requests": requests, "past": past, "new": new, "heads": heads, "group": group, "head_dim": head_dim, "block": block,
            "dtype": dtype, "causal": causal, "window": window, "ragged": ragged}


def listed():
    return [
        # queries and keys of a 21 x 30 x 52 video latent (12 heads of 128): time, height and width each with a ladder of its own
        {"name": "rotary_video_32760", **rotary_case(32760, 12, 12, 128, (22, 21, 21))},
        # a decode step of 16 requests deep in their contexts, one ladder cut into three sections, halves of a head rotated: latency
        {"name": "rotary_decode_16", **rotary_case(16, 40, 8, 128, (16, 24, 24), ladder="joint", style="halves", far=1_000_000)},
        # the gradient of an image tower's rotation (height and width), in FP32, an odd number of patches, part of a head rotated
        {"name": "rotary_image_inverse_4099", **rotary_case(4099, 16, 16, 64, (12, 12), dtype="fp32", style="halves", inverse=True, packed=False)},
        # one decode step of 256 requests: integers only, all latency
        {"name": "plan_decode_256", **plan_case(256, 16384, 1, 32, ragged=True)},
        # prompts of many lengths admitted at once
        {"name": "plan_prompts_40", **plan_case(40, 2048, 2500, 16, ragged=True)},
        # keys and values of a whole video latent
        {"name": "write_video_32760", **write_case(1, 0, 32760, 12, 128, 64)},
        # one decode step of 64 requests, appended in the middle of pages
        {"name": "write_decode_64", **write_case(64, 8192, 1, 8, 128, 32, dtype="fp16")},
        # one user's decode step after a long context: one token, 40 query heads on 8 key/value heads
        {"name": "decode_1x32760", **attention_case(1, 32760, 1, 8, 5, 128, 64)},
        # batched decode, contexts of many lengths, small pages
        {"name": "decode_64x8192", **attention_case(64, 8192, 1, 8, 8, 128, 16, dtype="fp16")},
        # prompts' next chunk, causal, heads of 64
        {"name": "chunk_6x1000", **attention_case(6, 3001, 1000, 4, 4, 64, 32, dtype="fp16")},
        # an autoregressive video model's next frame (30 x 52) over the frames before it: all of the frame's tokens see all
        {"name": "frame_1560_of_32760", **attention_case(1, 31200, 1560, 40, 1, 128, 128, causal=False, ragged=False)},
        # a whole video latent over itself
        {"name": "video_32760", **attention_case(1, 0, 32760, 12, 1, 128, 64, causal=False, ragged=False)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "plan", "write", "attention", "attention"])
    block = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 128, 256])
        axes = rng.choice([1, 2, 3])
        pairs = rng.choice([head_dim // 2, head_dim // 4])
        sections = [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)
        heads = rng.choice([1, 5, 8, 12, 40])
        return rotary_case(_log(rng, 1, 32760 * 1536 // (2 * heads * head_dim)) if heads * head_dim > 768 else _log(rng, 1, 32760), heads,
                           rng.choice([1, heads]), head_dim, sections, rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["axis", "joint"]),
                           rng.choice(["pairs", "halves"]), rng.random() < 0.3, rng.random() < 0.5, rng.choice([0, 5000, 1_000_000]))
    if op == "plan":
        requests = _log(rng, 1, 512)
        return plan_case(requests, _log(rng, 1, 16384), _log(rng, 1, max(1, 50000 // requests)), block, True, rng.random() < 0.3)
    if op == "write":
        requests, heads, head_dim = _log(rng, 1, 64), rng.choice([1, 3, 8, 12]), rng.choice([64, 128, 256])
        return write_case(requests, _log(rng, 1, 4096), _log(rng, 1, 32760 * 1536 // (requests * heads * head_dim * 2)), heads, head_dim, block,
                          rng.choice(["bf16", "fp16"]), True, rng.random() < 0.5)
    while True:
        c = attention_case(_log(rng, 1, 64), _log(rng, 1, 32760), rng.choice([1, 1, 2, 5, _log(rng, 1, 4096)]), rng.choice([1, 2, 8, 12]),
                           rng.choice([1, 4, 5, 8, 16]), rng.choice([64, 128, 256]), block, rng.choice(["bf16", "fp16"]), rng.random() < 0.7,
                           rng.choice([0, 0, 0, 1000]), True)
        w = work(c)
        tokens = sum(p + n for p, n in lengths(c))
        if w["flops"] < 1e12 and tokens * c["heads"] * c["head_dim"] < 4e8:
            return c


def lengths(c):
    """(cached tokens, new tokens) of every request."""
    if not c["ragged"]:
        return [(c["past"], c["new"])] * c["requests"]
    rng = random.Random("%d %d %d" % (c["requests"], c["past"], c["new"]))
    found = [(c["past"], c["new"])]
    for i in range(1, c["requests"]):
        found.append((rng.randint(c["past"] // 8, c["past"]), 0 if i % 8 == 7 else rng.randint(1 + c["new"] // 4, max(c["new"], 1 + c["new"] // 4))))
    return found


def _visible(c, past, new):
    """(row, key) pairs of one request and head, and the keys that some row sees."""
    total = past + new
    if not new:
        return 0, 0
    if not c["causal"]:
        low = max(0, past - c["window"] + 1) if c["window"] else 0
        pairs = sum(total - max(0, past + i - c["window"] + 1) for i in range(new)) if c["window"] else new * total
        return pairs, total - low
    if not c["window"]:
        return new * past + new * (new + 1) // 2, total
    return sum(min(past + i + 1, c["window"]) for i in range(new)), min(total, new + c["window"] - 1)


def work(case):
    c = case
    size = 4 if c.get("dtype") == "fp32" else 2
    if c["op"] == "rotary":
        values = c["tokens"] * (c["q_heads"] + c["k_heads"]) * c["head_dim"]
        return {"bytes": 2 * size * values + 4 * c["tokens"] * len(_sections(c)), "flops": 3 * values}
    every = lengths(c)
    tokens = sum(n for _, n in every)
    if c["op"] == "plan":
        pages = sum(-(-(p + n) // c["block"]) - -(-p // c["block"]) for p, n in every)
        return {"bytes": 12 * tokens + 16 * c["requests"] + 8 * pages, "flops": 0}
    if c["op"] == "write":
        values = 2 * c["heads"] * c["head_dim"]
        seen = sum(p % c["block"] + n for p, n in every if n)
        # new tokens in, codes out; the touched pages' codes in, their values out; of pages begun before, the scales and no more
        return {"bytes": values * (tokens * (size + 1) + seen * (1 + size)), "flops": 2 * values * (tokens + seen)}
    pairs, keys = (sum(v) for v in zip(*(_visible(c, p, n) for p, n in every)))
    q_heads = c["heads"] * c["group"]
    return {"bytes": 2 * size * tokens * q_heads * c["head_dim"] + 2 * keys * c["heads"] * c["head_dim"], "flops": 4 * pairs * q_heads * c["head_dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _sections(c):
    return [s for s in (c["s0"], c["s1"], c["s2"]) if s]


def _heads(g, tokens, heads, head_dim, dtype, spread=1.0):
    """Projected rows: most channels alike, a few with much larger values, each with an offset of its own."""
    gain = torch.ones(heads, head_dim, device=DEVICE)
    gain[:, :: max(1, head_dim // 3)] = 3.0
    mean = 0.4 * torch.randn(heads, head_dim, generator=g, device=DEVICE)
    x = torch.randn(tokens, heads, head_dim, generator=g, device=DEVICE)
    return (x.add_(mean).mul_(gain * spread)).to(dtype)


def _pages(c, g, total):
    """Pages of every request in the order of a used pool, as a table (requests, most pages), and the pages beyond them."""
    want = [-(-t // c["block"]) for t in total]
    pool = torch.randperm(sum(want) + 3, generator=g, device=DEVICE).int()
    tables = torch.zeros(len(total), max(1, *want), dtype=torch.int32, device=DEVICE) if len(want) > 1 else torch.zeros(1, max(1, want[0]), dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(want):
        tables[i, :n] = pool[at:at + n]
        at += n
    return tables, pool[at:]


def _codes(g, pages, heads, block, head_dim):
    """A cache that holds earlier tokens: codes (pages, heads, block, head_dim) int8 and scales (pages, heads)."""
    codes = torch.empty(pages, heads, block, head_dim, dtype=torch.int8, device=DEVICE)
    scales = torch.empty(pages, heads, device=DEVICE)
    mean = 0.4 * torch.randn(heads, 1, head_dim, generator=g, device=DEVICE)
    step = max(1, (1 << 27) // (heads * block * head_dim))
    for at in range(0, pages, step):
        x = torch.randn(min(step, pages - at), heads, block, head_dim, generator=g, device=DEVICE).add_(mean)
        x[..., :: max(1, head_dim // 3)] *= 3.0
        s = x.abs().amax((2, 3)) / 127
        scales[at:at + step] = s
        codes[at:at + step] = torch.round(x / s[..., None, None])
    return codes, scales


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _inputs(c, seed):
    g = _generator(seed)
    s = {"case": c}
    if c["op"] == "rotary":
        d, t, (qh, kh) = DTYPES[c["dtype"]], c["tokens"], (c["q_heads"], c["k_heads"])
        if c["packed"]:  # views of one projection's rows [q | k | v]
            rows = _heads(g, t, qh + 2 * kh, c["head_dim"], d)
            s["q"], s["k"] = rows[:, :qh], rows[:, qh:qh + kh]
        else:
            s["q"], s["k"] = _heads(g, t, qh, c["head_dim"], d), _heads(g, t, kh, c["head_dim"], d)
        axes = len(_sections(c))
        if c["far"]:
            s["positions"] = torch.randint(0, c["far"], (t, axes), generator=g, device=DEVICE, dtype=torch.int32)
        else:  # a grid, its fastest axis last
            index = torch.arange(t, device=DEVICE) + int(torch.randint(0, 1000, (1,), generator=g, device=DEVICE))
            grid = [index] if axes == 1 else [index // 52, index % 52] if axes == 2 else [index // 1560, index // 52 % 30, index % 52]
            s["positions"] = torch.stack(grid, 1).int()
        return s
    every = lengths(c)
    s["lengths"], s["tokens"] = every, sum(n for _, n in every)
    if c["op"] == "plan":
        # lengths move with the seed here: they are the inputs
        rng = random.Random(seed)
        width = max(-(-(p + n) // c["block"]) for p, n in every) + 1
        every = [(max(0, p - rng.randint(0, min(p, 40))), n) for p, n in every]
        have = [-(-p // c["block"]) for p, _ in every]
        want = [-(-(p + n) // c["block"]) for p, n in every]
        need = sum(want) - sum(have)
        pool = torch.randperm(sum(have) + need + 50, generator=g, device=DEVICE).int()
        s["tables"] = torch.full((len(every), width), -1, dtype=torch.int32, device=DEVICE)
        at = 0
        for i, n in enumerate(have):
            s["tables"][i, :n] = pool[at:at + n]
            at += n
        taken = rng.randint(0, 40)
        s["free"] = torch.cat([pool[:taken], pool[at:at + (need * 2 // 3 if c["tight"] else need + 5)]])
        s["used"] = _ints([taken])
        s["past"], s["new"] = _ints([p for p, _ in every]), _ints([n for _, n in every])
        return s
    total = [p + n for p, n in every]
    s["tables"], spare = _pages(c, g, total)
    pages = int(sum(-(-t // c["block"]) for t in total)) + 3
    s["codes"] = [_codes(g, pages, c["heads"], c["block"], c["head_dim"]) for _ in range(2)]
    d = DTYPES[c["dtype"]]
    if c["op"] == "write":
        h = c["heads"]
        if c["packed"]:
            rows = _heads(g, s["tokens"], 2 * h, c["head_dim"], d)
            s["k"], s["v"] = rows[:, :h], rows[:, h:]
        else:
            s["k"], s["v"] = _heads(g, s["tokens"], h, c["head_dim"], d), _heads(g, s["tokens"], h, c["head_dim"], d)
        index = [(i, torch.arange(p, p + n)) for i, (p, n) in enumerate(every)]
        slot = lambda i, at: s["tables"][i, (at // c["block"]).to(DEVICE)].long() * c["block"] + (at % c["block"]).to(DEVICE)
        s["slots"] = torch.cat([slot(i, at) for i, at in index])
        s["seen"] = torch.cat([slot(i, torch.arange(p // c["block"] * c["block"], p + n)) if n else slot(i, torch.arange(0)) for i, (p, n) in enumerate(every)])
        return s
    s["q"] = _heads(g, s["tokens"], c["heads"] * c["group"], c["head_dim"], d, 0.8)
    s["lens"] = _ints(total)
    s["starts"] = _ints([0] + list(np.cumsum([n for _, n in every])))
    return s


def prepare(case, seed):
    c = {k: v for k, v in case.items() if k != "name"}
    s = _inputs(c, seed)
    if own:
        from wgpkernels_amd import int8
        s["int8"] = int8
        int8.library()
        if c["op"] == "rotary":
            s["plan"] = int8.rotary_plan(_sections(c), ladder=c["ladder"], style=c["style"], device=DEVICE)
        elif c["op"] in ("write", "attention"):
            (k, ks), (v, vs) = s.pop("codes")
            s["cache"] = int8.KVCache.from_codes(k, ks, v, vs)
    elif c["op"] == "rotary":
        s["frequencies"], s["axis"] = (t.to(DEVICE) for t in _ladder(c))
    elif c["op"] == "write":
        s["runs"] = _runs(c, s)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _ladder(c):
    """Frequency (64 bits) and axis of every rotated pair."""
    sections = _sections(c)
    pairs = sum(sections)
    steps = [torch.arange(n, dtype=torch.float64) / n for n in sections] if c["ladder"] == "axis" else [torch.arange(pairs, dtype=torch.float64) / pairs]
    return 10000.0 ** -torch.cat(steps), torch.cat([torch.full((n,), a) for a, n in enumerate(sections)])


def _rotate_plain(x, cos, sin, style):
    r, out = 2 * cos.shape[-1], x.float().clone()
    f = out[..., :r]
    a, b = (f[..., 0::2], f[..., 1::2]) if style == "pairs" else f.chunk(2, -1)
    a, b = a * cos - b * sin, a * sin + b * cos
    out[..., :r] = torch.stack([a, b], -1).flatten(-2) if style == "pairs" else torch.cat([a, b], -1)
    return out.to(x.dtype)


def _rotary_plain(s):
    c = s["case"]
    angle = s["positions"].double()[:, s["axis"]] * s["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    sin = -sin if c["inverse"] else sin
    return {"q": _rotate_plain(s["q"], cos, sin, c["style"]), "k": _rotate_plain(s["k"], cos, sin, c["style"])}


def _plan_plain(s):
    c, block, width, tokens = s["case"], s["case"]["block"], s["tables"].shape[1], s["tokens"]
    past, new, used = s["past"].clamp(min=0).long(), s["new"].clamp(min=0).long(), s["used"].long()
    have, want = (past + block - 1) // block, (past + new + block - 1) // block
    ends = new.cumsum(0)
    starts = ends - new
    fits = (want <= width) & (ends <= tokens)
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (used + upto <= s["free"].shape[0]))
    column = torch.arange(width, device=DEVICE)
    fresh = ok[:, None] & (column >= have[:, None]) & (column < want[:, None])
    source = (used + (upto - need)[:, None] + column - have[:, None]).clamp(0, max(0, s["free"].shape[0] - 1))
    s["tables"].copy_(torch.where(fresh, s["free"][source], s["tables"]))
    token = torch.arange(tokens, device=DEVICE)
    row = torch.searchsorted(ends, token, right=True)
    inside = row < len(past)
    row = row.clamp(max=len(past) - 1)
    position = past[row] + token - starts[row]
    page = s["tables"][row, (position // block).clamp(max=width - 1)].long()
    slots = torch.where(inside & ok[row], page * block + position % block, -1)
    return {"tables": s["tables"], "slots": slots, "positions": torch.where(inside, position, 0).int(),
            "starts": torch.cat([starts[:1], ends]).clamp(max=tokens).int(), "lens": torch.where(ok, past + new, past).int(),
            "used": (used + torch.where(ok, need, 0).sum()).int(), "missing": (~ok).sum().int()[None]}


def _runs(c, s):
    """The touched pages: page, tokens that it held, and its new tokens' rows (pages, block; -1: none of them)."""
    block, slots = c["block"], s["slots"]
    pages, run = torch.unique_consecutive(slots // block, return_inverse=True)
    rows = torch.full((len(pages), block), -1, dtype=torch.long, device=DEVICE)
    rows[run, slots % block] = torch.arange(len(slots), device=DEVICE)
    return pages, (rows >= 0).int().argmax(1), rows


def _write_plain(x, codes, scales, runs):
    pages, held, rows = runs
    fresh = rows >= 0
    values = torch.where(fresh[..., None, None], x[rows.clamp(min=0)].float(), 0.0)  # (pages, block, heads, head_dim)
    old = torch.where(held[:, None] > 0, scales[pages], 0.0)
    new = torch.maximum(old, values.abs().amax((1, 3)) / 127)
    by = torch.where(new > 0, new, 1.0).double()[:, :, None, None]
    coded = torch.round(values.transpose(1, 2).double() / by)
    before = codes[pages]
    again = torch.round(before.double() * old.double()[:, :, None, None] / by)
    earlier = torch.arange(rows.shape[1], device=DEVICE) < held[:, None]
    out = torch.where(fresh[:, None, :, None], coded, torch.where(earlier[:, None, :, None], again, before.double()))
    codes[pages], scales[pages] = out.to(torch.int8), new


def _read_plain(codes, scales, slots, dtype):
    block = codes.shape[2]
    page, at = slots // block, slots % block
    return (codes[page, :, at].float() * scales[page][..., None]).to(dtype)


def _attention_plain(s):
    c, out = s["case"], torch.empty_like(s["q"])
    block, h, group, d = c["block"], c["heads"], c["group"], c["head_dim"]
    at = 0
    for i, (past, new) in enumerate(s["lengths"]):
        total = past + new
        if not new:
            continue
        pages = s["tables"][i, :-(-total // block)].long()
        k, v = ((codes[pages].float() * scales[pages][..., None, None]).transpose(0, 1).reshape(h, -1, d)[:, :total] for codes, scales in s["codes"])
        # rows (head, token and group, head_dim) on keys (head, token, head_dim)
        q = s["q"][at:at + new].float().reshape(new, h, group, d).permute(1, 0, 2, 3).reshape(h, new * group, d)
        o = torch.empty_like(q)
        heads = max(1, (1 << 31) // (new * group * total))
        rows = max(1, (1 << 31) // total)
        key = torch.arange(total, device=DEVICE)
        for a in range(0, h, heads):
            kt, va = k[a:a + heads].transpose(1, 2).contiguous(), v[a:a + heads]
            for b in range(0, new * group, rows):
                scores = torch.bmm(q[a:a + heads, b:b + rows], kt).mul_(d ** -0.5)
                position = past + torch.arange(b, min(b + rows, new * group), device=DEVICE)[:, None] // group
                if c["causal"]:
                    scores.masked_fill_(key > position, -math.inf)
                if c["window"]:
                    scores.masked_fill_(key <= position - c["window"], -math.inf)
                scores.sub_(scores.amax(-1, keepdim=True)).exp_()
                o[a:a + heads, b:b + rows] = torch.bmm(scores, va) / scores.sum(-1, keepdim=True)
        out[at:at + new] = o.reshape(h, new, group, d).permute(1, 0, 2, 3).reshape(new, h * group, d).to(out.dtype)
        at += new
    return {"out": out}


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "rotary":
            return _rotary_plain(s)
        if c["op"] == "plan":
            return _plan_plain(s)
        if c["op"] == "write":
            for x, (codes, scales) in zip((s["k"], s["v"]), s["codes"]):
                _write_plain(x, codes, scales, s["runs"])
            k, v = (_read_plain(*held, s["seen"], s["k"].dtype) for held in s["codes"])
            return {"k": k, "v": v}
        return _attention_plain(s)
    wq = s["int8"]
    if c["op"] == "rotary":
        q, k = wq.rotary((s["q"], s["k"]), s["positions"], s["plan"], inverse=c["inverse"])
        return {"q": q, "k": k}
    if c["op"] == "plan":
        p = wq.kv_plan(s["past"], s["new"], s["tables"], s["free"], s["used"], c["block"], s["tokens"])
        return {"tables": s["tables"], "slots": p.slots, "positions": p.positions, "starts": p.starts, "lens": p.lens, "used": p.used, "missing": p.missing}
    if c["op"] == "write":
        wq.kv_write(s["cache"], s["k"], s["v"], s["slots"])
        k, v = wq.kv_read(s["cache"], s["seen"], s["k"].dtype)
        return {"k": k, "v": v}
    return {"out": wq.kv_attention(s["q"], s["cache"], s["tables"], s["lens"], s["starts"], causal=c["causal"], window=c["window"])}


# ---- 64 bits, from the definitions ----------------------------------------------------------------------------------
def _exact_rotary(c, s):
    sections, style = _sections(c), c["style"]
    pairs, found = sum(sections), {}
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if style == "pairs" else torch.complex(x[..., :pairs], x[..., pairs:2 * pairs])
        at = 0
        for a, n in enumerate(sections):
            exponent = torch.arange(n, dtype=torch.float64, device=DEVICE) / n if c["ladder"] == "axis" else torch.arange(at, at + n, dtype=torch.float64, device=DEVICE) / pairs
            angle = torch.outer(s["positions"][:, a].double(), torch.exp(-math.log(10000.0) * exponent))
            z[..., at:at + n] *= torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)[:, None]
            at += n
        if style == "pairs":
            x[..., :2 * pairs] = torch.view_as_real(z).flatten(-2)
        else:
            x[..., :pairs], x[..., pairs:2 * pairs] = z.real, z.imag
        found[name] = x
    return found


def _exact_write(c, s):
    """Every page on its own, from the rows that its slots name."""
    found, block = {}, c["block"]
    slots, seen = s["slots"], s["seen"]
    order = torch.argsort(slots)
    page, count = torch.unique_consecutive(slots[order] // block, return_counts=True)
    owner = torch.repeat_interleave(torch.arange(len(page), device=DEVICE), count)
    first = torch.zeros_like(count).scatter_reduce(0, owner, slots[order] % block, "amin", include_self=False)
    for name, x, (codes, scales) in zip("kv", (s["k"], s["v"]), s["codes"]):
        x = x[order].double()
        top = torch.zeros(len(page), c["heads"], dtype=torch.float64, device=DEVICE)
        top = top.scatter_reduce(0, owner[:, None].expand(-1, c["heads"]), x.abs().amax(-1), "amax")
        fresh = (top / 127).float().double()  # a scale is held in FP32
        held = scales.double()[page] * (first > 0)[:, None]
        scale = torch.maximum(fresh, held)
        where = torch.searchsorted(page, seen // block)
        s_of, h_of = scale[where][..., None], held[where][..., None]
        old = codes[seen // block, :, seen % block].double()
        value = torch.round(old * h_of / s_of) * s_of
        sorted_slots = slots[order]
        at = torch.searchsorted(sorted_slots, seen).clamp(max=len(slots) - 1)
        mine = sorted_slots[at] == seen
        value[mine] = torch.round(x[at[mine]] / s_of[mine]) * s_of[mine]
        found[name] = value
    return found


def _exact_attention(c, s):
    """Key blocks one after another, with the running maximum and sums, each row's keys chosen by their slots."""
    block, h, group, d = c["block"], c["heads"], c["group"], c["head_dim"]
    (kc, ks), (vc, vs) = s["codes"]
    parts, at = [], 0
    for i, (past, new) in enumerate(s["lengths"]):
        total = past + new
        if not new:
            continue
        q = (s["q"][at:at + new].double() * d ** -0.5).unflatten(1, (h, group)).permute(1, 2, 0, 3).reshape(h, group * new, d)
        row = past + torch.arange(new, device=DEVICE).repeat(group)[:, None]
        at += new
        top = torch.full((h, group * new, 1), -math.inf, dtype=torch.float64, device=DEVICE)
        mass, acc = torch.zeros_like(top), torch.zeros_like(q)
        step = max(block, min(8192, (1 << 28) // (h * group * new)) // block * block)
        for low in range(0, total, step):
            key = torch.arange(low, min(total, low + step), device=DEVICE)
            page, off = s["tables"][i, key // block].long(), key % block
            k = (kc[page, :, off].double() * ks.double()[page][..., None]).permute(1, 2, 0).contiguous()
            v = (vc[page, :, off].double() * vs.double()[page][..., None]).transpose(0, 1).contiguous()
            hidden = torch.zeros(group * new, len(key), dtype=torch.bool, device=DEVICE)
            if c["causal"]:
                hidden |= key[None] > row
            if c["window"]:
                hidden |= key[None] <= row - c["window"]
            score = torch.bmm(q, k).masked_fill_(hidden, -math.inf)
            higher = torch.maximum(top, score.amax(-1, keepdim=True))
            safe = torch.where(higher.isinf(), 0.0, higher)
            keep, weight = torch.exp(top - safe), torch.exp(score - safe)
            mass, acc, top = mass * keep + weight.sum(-1, keepdim=True), acc * keep + torch.bmm(weight, v), higher
        parts.append((acc / mass).reshape(h, group, new, d).permute(2, 0, 1, 3).reshape(new, h * group, d))
    return {"out": torch.cat(parts)}


def exact(case, seed):
    c = {k: v for k, v in case.items() if k != "name"}
    if c["op"] == "plan":
        return None
    s = _inputs(c, seed)
    return {"rotary": _exact_rotary, "write": _exact_write, "attention": _exact_attention}[c["op"]](c, s)
