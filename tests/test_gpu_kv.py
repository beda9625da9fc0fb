"""The 8-bit key/value cache on the GPU: plans against a plain walk over the requests, writes and reads against 64 bits.

Tolerance of a held value: half a step of its page's scale, and 2^-14 of a step for the FP32 quotient (|quotient| <= 127, within
2^-23 of itself, twice: 127 * 2^-22 < 2^-14); a token that is coded again after its page's scale grew is off by as much again from
what it was. Reads round code * scale once: half a step of the type."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ---- plans ---------------------------------------------------------------------------------------------------------
def walk(past, new, tables, free, used, block, tokens):
    """The plan, one request after another."""
    tables = [list(row) for row in tables]
    width, taken, asked = len(tables[0]) if tables else 0, used, used
    slots, positions, starts, lens, missing = [], [], [0], [], 0
    for r, (p, n) in enumerate(zip(past, new)):
        p, n = max(0, p), max(0, n)
        have, want = -(-p // block), -(-(p + n) // block)
        end = starts[-1] + n if r else n
        end = sum(max(0, v) for v in new[:r + 1])
        fits = want <= width and end <= tokens
        asked += want - have if fits else 0
        ok = fits and (want == have or asked <= len(free))
        if ok:
            tables[r][have:want] = free[asked - (want - have):asked]
            taken += want - have
        missing += not ok
        starts.append(min(end, tokens))
        lens.append(p + n if ok else p)
        for i in range(p, p + n):
            if len(slots) < tokens:
                slots.append(tables[r][i // block] * block + i % block if ok else -1)
                positions.append(i)
    pad = tokens - len(slots)
    return tables, slots + [-1] * pad, positions + [0] * pad, starts, lens, [taken], [missing]


@pytest.mark.parametrize("requests,most_past,most_new,block,room", [(1, 0, 1, 16, 5), (1, 100, 5000, 64, 5), (3, 40, 70, 16, -4), (64, 300, 1, 32, 3),
                                                                    (257, 60, 9, 16, 0), (600, 30, 30, 16, -200), (40, 900, 400, 128, 9), (5, 20, 20, 7, 2)])
def test_plan(wq, requests, most_past, most_new, block, room):
    print(f"plan {requests} {most_past} {most_new} {block} {room}", flush=True)
    rng = random.Random(requests)
    past = [rng.randint(0, most_past) for _ in range(requests)]
    new = [rng.choice([0, rng.randint(0, most_new), most_new]) for _ in range(requests)]
    past[0], new[-1] = max(past[0] - 1, 0), -3 if requests > 2 else new[-1]
    width = max(-(-(p + max(n, 0)) // block) for p, n in zip(past, new)) + (1 if requests != 40 else -1)
    need = sum(-(-(p + max(n, 0)) // block) - -(-p // block) for p, n in zip(past, new))
    pages = list(range(10, 10 + need + 4000))
    rng.shuffle(pages)
    tables = [[pages.pop() if c < -(-p // block) else -1 for c in range(width)] for p in past]
    used = 3
    free = pages[:used + max(0, need + room)]
    total = sum(max(0, n) for n in new)
    for tokens in (total, total + 11, max(0, total - 5)):
        want = walk(past, new, tables, free, used, block, tokens)
        wide = torch.full((requests, width + 3), -7, dtype=torch.int32, device="cuda")  # rows of a larger table
        held = wide[:, :width]
        held.copy_(ints(tables))
        got = wq.kv_plan(ints(past), ints(new), held, ints(free), ints([used]), block, tokens)
        for name, a, b in zip(("tables", "slots", "positions", "starts", "lens", "used", "missing"),
                              (held, got.slots, got.positions, got.starts, got.lens, got.used, got.missing), want):
            assert a.tolist() == b, name
        assert (wide[:, width:] == -7).all()


def test_plan_at_the_last_positions(wq):
    """Positions end at 2^31 - 1: a request that would pass them finds no room."""
    last = 2 ** 31 - 1
    tables = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    past, new = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([last - 3, last - 2], [3, 3]))
    plan = wq.kv_plan(past, new, tables, torch.arange(4, device="cuda").int(), torch.zeros(1, dtype=torch.int32, device="cuda"), 2 ** 30, 6)
    assert plan.lens.tolist() == [last, last - 2] and plan.missing.tolist() == [1]
    assert plan.positions[:3].tolist() == [last - 3, last - 2, last - 1] and plan.slots[:3].tolist() == [2 ** 30 - 4, 2 ** 30 - 3, 2 ** 30 - 2]
    assert plan.slots[3:].tolist() == [-1] * 3


def test_plan_of_nothing(wq):
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    plan = wq.kv_plan(none, none, none.reshape(0, 4), none, ints([2]), 16, 3)
    assert plan.slots.tolist() == [-1] * 3 and plan.starts.tolist() == [0] and plan.used.tolist() == [2] and plan.missing.tolist() == [0]
    plan = wq.kv_plan(ints([5]), ints([0]), ints([[1, 2]]), none, ints([0]), 16, 0)
    assert plan.slots.shape == (0,) and plan.lens.tolist() == [5] and plan.starts.tolist() == [0, 0]


# ---- writes and reads ----------------------------------------------------------------------------------------------
def step_of(scale):
    return scale.double() * (0.5 + 2.0 ** -14)


def held(cache, which):
    codes, scales = (cache.k_codes, cache.k_scales) if which == "k" else (cache.v_codes, cache.v_scales)
    return codes.double() * scales.double()[..., None, None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,head_dim,block", [(1, 1, 64, 16), (5, 3, 128, 32), (300, 2, 256, 16), (513, 1, 64, 128), (700, 3, 128, 64), (1500, 2, 72, 16)])
@pytest.mark.parametrize("order", ["run", "any"])
def test_write(wq, dtype, tokens, heads, head_dim, block, order):
    """Runs of tokens, or slots in any order with holes: new values and scales, what the pages held before, and what is left alone."""
    print(f"write {dtype} {tokens} {heads} {head_dim} {block} {order}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = -(-tokens // block) + 3
    cache = wq.KVCache(pages, heads, head_dim, block)
    cache.owner.random_(0, tokens + 5, generator=g)  # scratch of earlier calls
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.random_(-127, 128, generator=g)
        scales.uniform_(0.001, 0.03, generator=g)  # some grow, some do not
    if order == "run":
        slots = torch.arange(tokens, device="cuda") + block // 2 + 1
    else:
        slots = torch.randperm(pages * block, generator=g, device="cuda")[:tokens]
        slots[::7] = -1
    wide = torch.randn(tokens, 2 * heads + 1, head_dim, generator=g, device="cuda").to(dtype)
    k, v = wide[:, :heads], wide[:, heads + 1:]
    before = {n: held(cache, n) for n in "kv"}
    old = {n: (getattr(cache, n + "_codes").clone(), getattr(cache, n + "_scales").clone()) for n in "kv"}
    wq.kv_write(cache, k, v, slots)
    live = slots >= 0
    page, at = slots[live] // block, slots[live] % block
    fresh = torch.zeros(pages, block, dtype=torch.bool, device="cuda")
    fresh[page, at] = True
    for n, x in (("k", k), ("v", v)):
        now, scales = held(cache, n), getattr(cache, n + "_scales")
        values = torch.zeros(pages, block, heads, head_dim, dtype=torch.float64, device="cuda")
        values[page, at] = x[live].double()
        anew = fresh[:, :1]
        start = torch.where(anew, 0.0, old[n][1])
        want = torch.maximum(start, (values.abs().amax((1, 3)) / 127).float())
        assert torch.equal(scales, torch.where(fresh.any(1)[:, None], want, old[n][1]))
        assert ((now[page, :, at] - x[live].double()).abs() <= step_of(scales)[page][..., None]).all()
        kept = ~fresh & ~anew  # held by a page that goes on
        off = (now - before[n]).abs().amax(3).transpose(1, 2)  # (pages, block, heads)
        assert (off <= torch.where(scales > old[n][1], step_of(scales), 0.0)[:, None])[kept].all()
    # read back, rounded once
    asked = torch.cat([slots, ints([pages * block, -1, 0], torch.int64)])
    for out in (dtype, torch.float32):
        for got, n in zip(wq.kv_read(cache, asked, out), "kv"):
            inside = (asked >= 0) & (asked < pages * block)
            want = torch.where(inside[:, None, None], held(cache, n)[asked.clamp(0, pages * block - 1) // block, :, asked.clamp(0) % block], 0.0)
            step = torch.finfo(out).eps / 2
            assert ((got.double() - want).abs() <= step * want.abs() + torch.finfo(out).smallest_normal * step).all()


def test_growing_page(wq):
    """One token after another onto one page, each larger than the last: every token stays within a step of what it was."""
    cache = wq.KVCache(2, 1, 64, 16)
    cache.k_scales.fill_(5.0)  # an earlier owner's
    x = torch.randn(16, 1, 64, device="cuda") * torch.arange(1, 17, device="cuda")[:, None, None]
    for t in range(16):
        wq.kv_write(cache, x[t:t + 1], x[t:t + 1], ints([16 + t], torch.int64))
    scale = (x.abs().max().double() / 127).float()
    assert cache.k_scales[1].item() == scale.item() and cache.k_scales[0].item() == 5.0
    off = (held(cache, "k")[1, 0] - x[:, 0].double()).abs().amax(1)
    grown = torch.tensor([len({x[:j + 1].abs().max().item() for j in range(t, 16)}) for t in range(16)], device="cuda")
    assert (off <= step_of(scale) * grown).all()


def test_values_that_are_not_finite(wq):
    """NaN is held as zero, an infinity as the largest finite number; other heads and pages keep their values."""
    cache = wq.KVCache(3, 2, 64, 16)
    k = torch.randn(4, 2, 64, device="cuda").bfloat16()
    wq.kv_write(cache, k, k, ints([16, 17, 32, 33], torch.int64))
    good, before = wq.kv_read(cache, ints([16, 32, 33], torch.int64)), cache.k_scales.clone()
    bad = k[:2].clone()
    bad[0, 0, 5], bad[1, 1, 3] = math.nan, -math.inf
    wq.kv_write(cache, bad, bad, ints([18, 34], torch.int64))
    assert all(torch.isfinite(t).all() for t in (cache.k_scales, cache.v_scales))
    again = wq.kv_read(cache, ints([16, 32, 33], torch.int64))
    # where the new tokens' finite values made a scale grow, tokens were coded again: within half a step of what they were (and read in BF16)
    grown = torch.where(cache.k_scales > before, step_of(cache.k_scales), 0.0)
    for a, b in zip(good, again):
        off = (a.double() - b.double()).abs() - 2.0 ** -8 * (a.double().abs() + b.double().abs()) * (a != b)
        assert (off[:1] <= grown[1][:, None]).all() and (off[1:, 0] <= grown[2, 0]).all()
    k, _ = wq.kv_read(cache, ints([18, 34], torch.int64), torch.float32)
    assert k[0, 0, 5] == 0 and abs(k[1, 1, 3].item() / -torch.finfo(torch.float32).max - 1) < 2 ** -20


def test_small_and_zero_values(wq):
    for size in (0.0, 1e-42, 3e-39, 1e-30):
        cache = wq.KVCache(1, 1, 64, 16)
        x = torch.randn(3, 1, 64, device="cuda") * size
        wq.kv_write(cache, x, x, ints([0, 1, 2], torch.int64))
        scale = cache.k_scales[0, 0]
        # the scale itself is rounded, to 2^-149 where it is below 2^-126: up to 127 times half of that at the largest value
        assert ((held(cache, "k")[0, 0, :3] - x[:, 0].double()).abs() <= step_of(scale) + 127 * 2.0 ** -150).all()


def test_no_tokens(wq):
    cache = wq.KVCache(2, 1, 64, 16)
    none = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.empty(0, dtype=torch.int64, device="cuda")
    wq.kv_write(cache, none, none, slots)
    assert wq.kv_read(cache, slots)[0].shape == (0, 1, 64) and not cache.k_codes.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pages", [7, 70])
def test_codes_are_the_rounded_quotients(wq, dtype, pages):
    """16-bit values over their page's scale: the code is round(value / scale) in 64 bits, also of half the page's maximum, which is 63.5
    but for the rounding of the scale. Whole pages, and pages that go on under the scale of what they hold."""
    heads, d, block = 3, 64, 16
    g = torch.Generator(device="cuda").manual_seed(pages)
    x = torch.randn(pages, block, heads, d, generator=g, device="cuda").to(dtype)
    top = x.abs().amax((1, 3))
    x[:, 2, :, 9], x[:, 3, :, 1], x[:, 12, :, 30], x[:, 13, :, 31] = top, top / 2, top / 2, -top / 2
    x = x.reshape(pages * block, heads, d)
    slots = torch.arange(pages * block, device="cuda")
    cache = wq.KVCache(pages, heads, d, block)
    wq.kv_write(cache, x, x.neg(), slots)
    quotient = x.double() / cache.k_scales.double().repeat_interleave(block, 0)[..., None]
    assert (quotient.abs() - 63.5).abs().amin() < 2.0 ** -17 and torch.unique(torch.round(quotient).abs()).numel() > 100
    codes = lambda c: c.transpose(1, 2).reshape(pages * block, heads, d).double()
    assert torch.equal(codes(cache.k_codes), torch.round(quotient)) and torch.equal(codes(cache.v_codes), torch.round(-quotient))
    parts = wq.KVCache(pages, heads, d, block)
    first = slots % block < 8
    for some in (first, ~first):
        wq.kv_write(parts, x[some], x[some].neg(), slots[some])
    assert torch.equal(parts.k_scales, cache.k_scales) and torch.equal(parts.k_codes, cache.k_codes) and torch.equal(parts.v_codes, cache.v_codes)
