"""Attention over the 8-bit cache on the GPU against 64 bits.

Tolerance, for a row with weights p_j (summing to one) and values v_j of one channel: half a step of the output type of the value; for
the weights, held in FP16, half a step (2^-11) of sum p |v|, and as much again for the scores (FP32 sums of 128 products of
sum |q k| scale <= 64 or 256 of <= 32: off by 2^-11 at most, each weight by that share); for weights below FP16's normal range, half its
smallest step, 2^-25, of every key at the largest value (weights are relative to the largest weight times scale, so that no
page's scale enters)."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(wq, lens, heads, head_dim, block, seed=0, spare=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    want = [-(-n // block) for n in lens]
    pages = sum(want) + spare
    cache = wq.KVCache(pages, heads, head_dim, block)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.random_(-127, 128, generator=g)
        scales.uniform_(0.004, 0.03, generator=g)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    tables = torch.full((len(lens), max(1, *want, 1) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(want):
        tables[r, :n] = order[at:at + n]
        at += n
    return cache, tables


def exact(q, cache, tables, lens, new, causal, window, scale=None):
    """Rows, the bound's sum p |v|, and 2^-25 n max |v| over the row's weight sum."""
    q = q.cpu().double()
    heads, block, d = cache.heads, cache.block, cache.head_dim
    group = q.shape[1] // heads
    out, size, small = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    k_all, v_all = ((c.cpu().double() * s.cpu().double()[..., None, None]) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    for r, (n, m) in enumerate(zip(lens, new)):
        table = tables[r].cpu()
        keys = [j for j in range(min(n, table.shape[0] * block)) if 0 <= table[j // block] < cache.pages]
        page, off = table[[j // block for j in keys]].long(), torch.tensor([j % block for j in keys], dtype=torch.long)
        k, v = (x[page, :, off] for x in (k_all, v_all))  # (keys, heads, d)
        position = torch.tensor(keys)
        for t in range(m):
            own = n - m + t
            seen = torch.ones(len(keys), dtype=torch.bool)
            if causal:
                seen &= position <= own
            if window:
                seen &= position > own - window
            if not seen.any():
                continue
            ks, vs = k[seen].repeat_interleave(group, 1), v[seen].repeat_interleave(group, 1)
            s = (ks * q[at + t]).sum(-1) * (d ** -0.5 if scale is None else scale)
            p = torch.softmax(s, 0)[..., None]
            out[at + t] = (p * vs).sum(0)
            size[at + t] = (p * vs.abs()).sum(0)
            small[at + t] = len(ks) * 2.0 ** -25 * vs.abs().amax((0, 2))[:, None]
        at += m
    return out, size, small


def check(got, q, cache, tables, lens, new, causal=True, window=0, scale=None):
    want, size, small = exact(q, cache, tables, lens, new, causal, window, scale)
    rows = sum(new)
    off = (got[:rows].cpu().double() - want[:rows]).abs()
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * want.abs().clamp(min=info.smallest_normal) + 2.0 ** -10 * size + small
    assert (off <= bound[:rows]).all(), (off / bound[:rows].clamp(min=1e-300)).max().item()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(new):
    return ints([sum(new[:i]) for i in range(len(new) + 1)])


def rows(tokens, q_heads, head_dim, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(tokens, q_heads, head_dim, generator=g, device="cuda") * (0.4 * 64 / head_dim)).to(dtype)


CASES = [  # lens, new tokens, heads, group, head_dim, block
    ([1], [1], 1, 1, 64, 16), ([0, 3], [0, 1], 2, 3, 128, 16), ([37], [1], 2, 5, 128, 32), ([2049], [1], 1, 8, 128, 64), ([700, 1, 0, 333], [1, 1, 0, 1], 2, 4, 64, 16),
    ([130, 64, 257], [2, 5, 3], 1, 16, 256, 128), ([90], [90], 2, 1, 64, 16), ([300, 17], [40, 17], 1, 4, 128, 32), ([513], [130], 2, 2, 256, 64),
    ([1000], [65], 1, 1, 128, 128), ([260, 5], [1, 5], 3, 7, 64, 64), ([1500] * 3, [1, 0, 1], 1, 1, 128, 16), ([4097], [2], 1, 12, 64, 128),
    ([65, 129, 193], [64, 1, 129], 1, 2, 128, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 50), (False, 33), (True, 1)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(wq, dtype, causal, window, case):
    lens, new, heads, group, head_dim, block = CASES[case]
    print(f"attention {dtype} causal={causal} window={window} {CASES[case]}", flush=True)
    cache, tables = make(wq, lens, heads, head_dim, block, case)
    q = rows(sum(new), heads * group, head_dim, dtype, case)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(new), causal=causal, window=window)
    check(got, q, cache, tables, lens, new, causal, window)


def test_strides_scale_and_padding(wq):
    """Queries and outputs inside wider rows, a scale of its own, rows of no request left alone."""
    lens, new = [70, 200], [3, 20]
    cache, tables = make(wq, lens, 2, 64, 32, 5)
    wide = rows(30, 9, 64, torch.bfloat16, 6)
    out = torch.full((30, 6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q, y = wide[:, 1:5], out[:, 2:]
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(new), scale=0.05, out=y)
    assert got is y and (out[:, :2] == 7).all() and (out[23:] == 7).all()
    check(y, q, cache, tables, lens, new, scale=0.05)


@pytest.mark.parametrize("new", [1, 70])
def test_rows_that_see_nothing(wq, new):
    """Lengths below the new tokens (a request that found no room keeps its old length), of zero, and tables of no page."""
    lens = [new // 2, 0, new]
    cache, tables = make(wq, [new, new, new], 1, 64, 16)
    q = rows(3 * new, 4, 64, torch.float16, 1)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new] * 3))
    check(got, q, cache, tables, lens, [new] * 3)
    assert not got[:new - new // 2].any() and not got[new:2 * new].any()
    none = wq.kv_attention(q, cache, tables[:, :0], ints(lens), starts_of([new] * 3))
    assert not none.any()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_cache_are_hidden(wq, new):
    lens = [400]
    cache, tables = make(wq, lens, 2, 128, 16)
    tables[0, 3], tables[0, 7], tables[0, 20] = -1, cache.pages, 2 ** 31 - 1
    q = rows(new, 4, 128, torch.bfloat16, 2)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]))
    check(got, q, cache, tables, lens, [new])
    tables.fill_(-5)
    assert not wq.kv_attention(q, cache, tables, ints(lens), starts_of([new])).any()


@pytest.mark.parametrize("new", [1, 40])
def test_lengths_beyond_the_table(wq, new):
    cache, tables = make(wq, [64], 1, 64, 16)
    q = rows(new, 2, 64, torch.bfloat16, 2)
    got = wq.kv_attention(q, cache, tables[:, :4], ints([70]), starts_of([new]))
    check(got, q, cache, tables[:, :4], [70], [new])


@pytest.mark.parametrize("new", [1, 50])
def test_scales_far_apart(wq, new):
    """Zero scales (pages of zeros), and keys and values of very different sizes, in either order."""
    lens = [640]
    cache, tables = make(wq, lens, 1, 64, 16, 9)
    used = tables[0, :40].long()
    for zero in (used[:5], used[17:18]):
        cache.k_scales[zero] = 0
        cache.k_codes[zero] = 0
        cache.v_scales[zero] = 0
        cache.v_codes[zero] = 0
    cache.v_scales[used[6:12]] *= 2.0 ** -13
    cache.v_scales[used[25:26]] *= 2.0 ** 9
    q = rows(new, 3, 64, torch.bfloat16, 4)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]))
    check(got, q, cache, tables, lens, [new])
    cache.v_scales.zero_()
    cache.v_codes.zero_()
    assert not wq.kv_attention(q, cache, tables, ints(lens), starts_of([new])).any()


@pytest.mark.parametrize("new", [1, 50])
def test_extreme_queries(wq, new):
    """Scores far apart (one key takes all), queries of FP16's and BF16's largest and smallest sizes; a NaN stays in its row."""
    lens = [300]
    cache, tables = make(wq, lens, 1, 64, 16, 11)
    for dtype, size in ((torch.float16, 200.0), (torch.bfloat16, 2.0 ** 100), (torch.bfloat16, 2.0 ** -100), (torch.float16, 2.0 ** -20)):
        q = (rows(new, 2, 64, torch.float32, 12) * size).to(dtype)
        scale = 64 ** -0.5 / max(1.0, size / 4)
        got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]), scale=scale)
        check(got, q, cache, tables, lens, [new], scale=scale)
    q = rows(new, 2, 64, torch.bfloat16, 12)
    clean = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]))
    q[new // 2, 1, 7] = math.nan
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]))
    assert torch.isnan(got[new // 2, 1]).all()
    got[new // 2, 1] = clean[new // 2, 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [1, 50])
def test_negative_scale(wq, dtype, new):
    lens = [400]
    cache, tables = make(wq, lens, 1, 64, 32, 13)
    q = rows(new, 3, 64, dtype, 14)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]), scale=-2.0)
    check(got, q, cache, tables, lens, [new], scale=-2.0)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("requests,new,window", [(70, 5, 0), (70, 5, 20), (1, 300, 0), (1, 300, 40)])
def test_large_values_that_a_row_does_not_see(wq, block, requests, new, window):
    """A page whose values are 2^100 times the others': rows before it, and those whose window has passed it, do not see it, and a page of zeros
    counts in all of them as any other. The requests share their pages."""
    length, heads = 640 + new // 2, 8 if requests > 1 else 1
    cache, tables = make(wq, [length], heads, 64, block, 15)
    tables = tables.repeat(requests, 1)
    zero = tables[0, 448 // block].long()
    cache.v_scales[zero] = 0
    cache.v_codes[zero] = 0
    lens, news = [length] * requests, [new] * requests
    q = rows(new * requests, 3 * heads, 64, torch.bfloat16, 16)
    for large in (640 // block, (length - new) // block, (length - 1) // block):
        kept = cache.v_scales.clone()
        cache.v_scales[tables[0, large].long()] *= 2.0 ** 100
        got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(news), window=window)
        check(got, q, cache, tables, lens, news, window=window)
        cache.v_scales.copy_(kept)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("large", [0, 1, 6, 9])
def test_values_further_apart_than_a_float_reaches(wq, block, new, large):
    """The small values' weights are in the sum, though 2^-128 of the largest product of weight and scale."""
    lens = [640]
    cache, tables = make(wq, lens, 2, 128, block, 17)
    cache.v_scales *= 2.0 ** -8
    cache.v_scales[tables[0, large].long()] *= 2.0 ** 120
    cache.v_scales[tables[0, large].long()] *= 2.0 ** 8
    q = rows(new, 4, 128, torch.bfloat16, 18)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of([new]))
    check(got, q, cache, tables, lens, [new])


def test_many_zero_values_before_others(wq):
    """24000 keys whose values are zero and whose weights are 2^7.5 of the first 128 keys', then a page of values: their share of the weights."""
    length, heads, requests = 24000, 8, 75
    cache = wq.KVCache(length // 16, heads, 64, 16)
    tables = torch.arange(length // 16, dtype=torch.int32, device="cuda").repeat(requests, 1)
    cache.k_codes[8:] = 1
    cache.k_scales.fill_(1.0)
    cache.k_scales[-1] = 2.0
    cache.v_codes[-1] = 100
    cache.v_scales[-1] = 0.01
    q = torch.ones(requests, heads, 64, dtype=torch.bfloat16, device="cuda")
    got = wq.kv_attention(q, cache, tables, ints([length] * requests), torch.arange(requests + 1, dtype=torch.int32, device="cuda"), scale=7.5 * math.log(2) / 64)
    most = 16 * 2.0 ** 15
    want = most / (most + (length - 144) * 2.0 ** 7.5 + 128)
    # half a step of the output and as much of the weights; the scale in FP32 times scores of 2^4: 2^-20
    assert (got.double() - want).abs().max() <= want * (2.0 ** -9 + 2.0 ** -11 + 2.0 ** -20)


def test_far_pages(wq):
    """Codes beyond 2^31 bytes from the cache's start."""
    pages = (2 ** 31 + 2 ** 29) // (2 * 128 * 128)
    cache = wq.KVCache(pages, 2, 128, 128)
    tables = ints([[pages - 1, 0, pages - 3, pages - 2]])
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(400, 2, 128, generator=g, device="cuda").bfloat16()
    slots = torch.cat([tables[0, i].long() * 128 + torch.arange(128, device="cuda") for i in range(4)])[:400]
    wq.kv_write(cache, k, k.neg(), slots)
    rk, rv = wq.kv_read(cache, slots)
    step = cache.k_scales[tables[0].long()].max().item()
    assert (rk.float() - k.float()).abs().max() <= step * 0.51 + 0.02 and torch.equal(rk, rv.neg())
    small = wq.KVCache(4, 2, 128, 128)  # the same on near pages
    wq.kv_write(small, k, k.neg(), torch.arange(400, device="cuda"))
    for new in (1, 60):
        q = rows(new, 8, 128, torch.bfloat16, 3)
        far = wq.kv_attention(q, cache, tables, ints([400]), starts_of([new]))
        near = wq.kv_attention(q, small, ints([[0, 1, 2, 3]]), ints([400]), starts_of([new]))
        assert torch.equal(far, near)


@pytest.mark.parametrize("requests,most,new", [(300, 40, 1), (520, 20, 3), (70, 900, 1)])
def test_many_requests(wq, requests, most, new):
    rng = random.Random(requests)
    news = [rng.randint(0, new) for _ in range(requests)]
    lens = [rng.randint(n, most) for n in news]
    cache, tables = make(wq, lens, 1, 64, 16, requests)
    q = rows(sum(news), 4, 64, torch.float16, 8)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(news))
    check(got, q, cache, tables, lens, news)


@pytest.mark.parametrize("lens,new", [([2500, 17, 900, 1, 0, 1700, 333, 64], [1] * 4 + [0] + [1] * 3), ([700] * 9, [1] * 9), ([40, 3000, 9], [1, 12, 1]),
                                      ([5000, 4999], [3, 2]), ([250] * 20 + [4000], [1] * 21)], ids=["ragged", "equal", "several tiles", "two", "one long"])
def test_few_tiles_over_many_workgroups(wq, lens, new):
    """Tiles that come apart into whole shares, and those that do not: no keys twice, none left out."""
    cache, tables = make(wq, lens, 2, 64, 32, len(lens))
    q = rows(sum(new), 2 * 3, 64, torch.float16, 23)
    got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(new))
    check(got, q, cache, tables, lens, new)


def test_same_bits_again_and_on_a_side_stream(wq):
    """Nothing depends on the order in which workgroups end."""
    lens, new = [3000, 40, 1700], [1, 30, 1]
    cache, tables = make(wq, lens, 2, 128, 32, 21)
    q = rows(32, 8, 128, torch.bfloat16, 22)
    first = wq.kv_attention(q, cache, tables, ints(lens), starts_of(new))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [wq.kv_attention(q, cache, tables, ints(lens), starts_of(new)) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, o) for o in others)


@pytest.mark.parametrize("new", [1, 40])
def test_step_in_a_graph(wq, new):
    """Plan, rotation, write and attention of a step captured once and replayed: requests grow by `new` tokens a replay, with eager work
    between the replays; each replay's outputs are those of the same calls made eagerly on a cache of their own."""
    requests, heads, group, d, block, room = 3, 2, 2, 64, 16, 40
    plan = wq.rotary_plan((32,), style="halves")
    g = torch.Generator(device="cuda").manual_seed(new)

    class Side:
        def __init__(self):
            self.cache = wq.KVCache(room, heads, d, block)
            self.tables = torch.full((requests, 12), -1, dtype=torch.int32, device="cuda")
            self.past, self.used = ints([0] * requests), ints([0])
            self.new, self.free = ints([new, new - 1, new]), torch.arange(room - 1, -1, -1, device="cuda").int()
            self.x = torch.empty(requests * new, heads * (group + 2), d, dtype=torch.bfloat16, device="cuda")

        def step(self):
            p = wq.kv_plan(self.past, self.new, self.tables, self.free, self.used, block, requests * new)
            q, k = wq.rotary((self.x[:, :heads * group], self.x[:, heads * group:heads * (group + 1)]), p.positions, plan)
            wq.kv_write(self.cache, k, self.x[:, heads * (group + 1):], p.slots)
            out = torch.zeros(q.shape, dtype=q.dtype, device="cuda")
            wq.kv_attention(q, self.cache, self.tables, p.lens, p.starts, out=out)
            self.past.copy_(p.lens)
            self.used.copy_(p.used)
            return out

    eager, captured = Side(), Side()
    captured.x.zero_()
    captured.step()  # kernels loaded outside the capture
    captured.past.zero_()
    captured.used.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step()
    captured.past.zero_()
    captured.used.zero_()
    for _ in range(4):
        x = torch.randn(eager.x.shape, generator=g, device="cuda").bfloat16()
        eager.x.copy_(x)
        captured.x.copy_(x)
        want = eager.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager.past, captured.past)
        assert torch.isfinite(out).all() and out.any()
