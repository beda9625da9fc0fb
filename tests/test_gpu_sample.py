"""sample() on the GPU against its definition on the CPU, weights as whole numbers of 2^-44 of the heaviest and sums as integers: the tokens are
whole numbers and have to be equal. (An exponential whose last bit differs moves a weight by one such part, and the token only where a draw
or top-p's border falls between: with these seeds it does not. Sums of FP64 weights would not do: half of 750 pairs is exactly a border.)"""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def defined(logits, draws, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row after another, from the definition."""
    found = []
    for row in range(len(logits)):
        of = lambda option: option[row].item() if isinstance(option, torch.Tensor) else torch.tensor(option).item()
        t, k, p, m = of(temperature), int(of(top_k)), of(top_p), of(min_p)
        l = logits[row].cpu().double()
        l = torch.where(l.isnan(), -math.inf, l)
        top = l.max()
        if top == -math.inf:
            found.append(-1)
            continue
        order = torch.sort(l, descending=True, stable=True).indices
        if not t > 0:
            found.append(order[0].item())
            continue
        weight = torch.where(l == top, 1.0, torch.exp(torch.where(l == top, 0.0, l - top) / t)) if top != math.inf else (l == top).double()
        share = weight
        weight = torch.round(weight * 2.0 ** 44).long()
        ordered = weight[order]
        kept = torch.ones(len(l), dtype=torch.bool)
        if 0 < k < len(l):
            kept[k:] = False
        if p < 1:
            mass = torch.cumsum(ordered * kept, 0)
            before = torch.cat([torch.zeros(1, dtype=torch.int64), mass[:-1]])
            kept &= before < math.ceil(Fraction(p) * mass[-1].item())
            kept[0] = True
        kept &= share[order] >= min(m, 1.0)
        left = torch.zeros_like(weight)
        left[order] = ordered * kept
        upto = torch.cumsum(left, 0)
        u = draws[row].item()
        u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
        found.append((upto > math.floor(Fraction(u) * upto[-1].item())).int().argmax().item())
    return torch.tensor(found)


def logits_of(rows, vocabulary, dtype, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(rows, vocabulary, generator=g, device="cuda") * spread
    likely = max(1, min(200, vocabulary // 4))
    at = torch.randint(0, vocabulary, (rows, likely), generator=g, device="cuda")
    l.scatter_add_(1, at, -torch.log(torch.rand(rows, likely, generator=g, device="cuda").clamp_(min=1e-6)) * 2)
    return l.to(dtype), torch.rand(rows, generator=g, device="cuda"), g


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocabulary", [(1, 1), (3, 2), (5, 7), (4, 255), (7, 2048), (3, 2049), (40, 1000), (1, 50001), (9, 33333), (2, 131072), (1100, 300), (2, 262144)])
@pytest.mark.parametrize("options", [{}, {"temperature": 0.6, "top_k": 40}, {"top_p": 0.9}, {"temperature": 1.7, "top_k": 30, "top_p": 0.8}, {"min_p": 0.1},
                                     {"top_k": 1}, {"temperature": 0.0}, {"temperature": 3.0, "top_p": 0.999, "min_p": 0.001}, {"top_k": 500, "top_p": 0.3}])
def test_tokens(wq, dtype, rows, vocabulary, options):
    print(f"sample {rows} {vocabulary} {dtype} {options}", flush=True)
    logits, draws, _ = logits_of(rows, vocabulary, dtype, seed=rows + vocabulary)
    tokens = wq.sample(logits, draws, **options)
    assert tokens.dtype == torch.int64
    assert torch.equal(tokens.cpu(), defined(logits, draws, **options))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocabulary", [777, 20011])
def test_every_row_its_own_options(wq, dtype, vocabulary):
    rows = 96
    logits, draws, g = logits_of(rows, vocabulary, dtype, seed=5)
    pick = lambda values, kind: torch.tensor(values, dtype=kind, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
    options = {"temperature": pick([0.0, -1.0, 0.3, 1.0, 2.0, 1e-30, 1e30, math.nan], FP32), "top_k": pick([0, -5, 1, 2, 50, 10 ** 6, vocabulary - 1], torch.int32),
               "top_p": pick([1.0, 2.0, 0.9, 0.5, 0.0, -1.0, 1e-30], FP32), "min_p": pick([0.0, 0.2, 1.0, 5.0, -1.0], FP32)}
    assert torch.equal(wq.sample(logits, draws, **options).cpu(), defined(logits, draws, **options))


@pytest.mark.parametrize("vocabulary", [5, 3000, 40000, 131072])
@pytest.mark.parametrize("options", [{}, {"top_k": 2}, {"top_k": 2500}, {"top_p": 0.5}, {"top_k": 20000, "top_p": 0.7}, {"top_p": 0.5, "min_p": 1.0}])
def test_equal_logits(wq, vocabulary, options):
    """All alike, and two values only: ties by the lowest index, more of them than the list of keys holds."""
    print(f"equal {vocabulary} {options}", flush=True)
    draws = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24], device="cuda")
    logits = torch.full((4, vocabulary), -3.5, device="cuda")
    assert torch.equal(wq.sample(logits, draws, **options).cpu(), defined(logits, draws, **options))
    logits[:, ::2] += 0.5
    logits = logits.to(BF16)
    assert torch.equal(wq.sample(logits, draws, **options).cpu(), defined(logits, draws, **options))


def test_many_near_logits(wq):
    """A flat FP32 row: tens of thousands of different keys in the bins of the cuts."""
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.rand(3, 100000, generator=g, device="cuda") * 1e-3
    draws = torch.rand(3, generator=g, device="cuda")
    for options in ({"top_k": 30001}, {"top_p": 0.31}, {"top_k": 60000, "top_p": 0.77}, {"top_k": 5}):
        assert torch.equal(wq.sample(logits, draws, **options).cpu(), defined(logits, draws, **options)), options


@pytest.mark.parametrize("options", [{}, {"top_k": 3}, {"top_p": 0.6}, {"temperature": 0.0}, {"min_p": 0.5}])
def test_masks_infinities_and_nan(wq, options):
    logits, draws, _ = logits_of(9, 5000, FP32, seed=8)
    inf, nan = math.inf, math.nan
    logits[0] = -inf
    logits[1] = nan
    logits[2] = -inf
    logits[2, 4321] = -1e30          # a mask that leaves one token, far below the others of its kind
    logits[3, 7:] = -inf
    logits[4, ::3] = nan
    logits[5, 100], logits[5, 200] = inf, inf
    logits[6] = torch.finfo(FP32).min
    logits[6, 17] = 0
    logits[7, 1:] = torch.finfo(FP32).min  # the type's lowest value as a mask
    logits[8] = torch.finfo(FP32).min
    tokens = wq.sample(logits, draws, **options).cpu()
    assert torch.equal(tokens, defined(logits, draws, **options))
    assert tokens[:3].tolist() == [-1, -1, 4321] and tokens[3] < 7 and tokens[4] % 3 and tokens[5] in (100, 200) and tokens[6] == 17 and tokens[7] == 0


def test_zeros_of_both_signs_are_alike(wq):
    logits = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device="cuda")
    for k in (1, 2, 3):
        draws = torch.tensor([1 - 2.0 ** -24], device="cuda")
        assert wq.sample(logits, draws, top_k=k).item() == k - 1
    assert wq.sample(logits, draws, temperature=0.0).item() == 0


def test_draws_at_the_ends_and_outside(wq):
    logits, _, _ = logits_of(6, 300, FP32, seed=3)
    logits[:, 0] = logits[:, 299] = 3.0
    draws = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan], device="cuda")
    assert wq.sample(logits, draws).tolist() == [0, 299, 299, 299, 0, 0]


def test_rows_apart_and_unaligned(wq):
    for dtype in (BF16, FP32):
        held, draws, _ = logits_of(5, 7001, dtype, seed=6)
        for first, last in ((1, 7000), (3, 4099), (5, 6)):
            view = held[:, first:last]
            for options in ({"top_k": 20, "top_p": 0.9}, {}):
                assert torch.equal(wq.sample(view, draws, **options).cpu(), defined(view, draws, **options))
        one = held[2, 1:].expand(4, 7000)  # the same row for several draws
        assert torch.equal(wq.sample(one, draws[:4].contiguous(), top_p=0.9).cpu(), defined(one, draws[:4], top_p=0.9))


def test_shares_follow_the_weights(wq):
    """Draws spread evenly over [0, 1): every token as often as its share says, but for one at each border."""
    logits = torch.log(torch.tensor([0.1, 0.4, 0.05, 0.25, 0.2], device="cuda"))
    n = 4096
    draws = (torch.arange(n, device="cuda").float() + 0.5) / n
    tokens = wq.sample(logits.expand(n, 5).contiguous(), draws)
    assert (tokens.bincount(minlength=5).cpu() - n * torch.softmax(logits.cpu(), 0)).abs().max() <= 1
    tokens = wq.sample(logits.expand(n, 5).contiguous(), draws, top_k=3)
    want = torch.tensor([0, 0.4, 0, 0.25, 0.2]) / 0.85 * n
    assert (tokens.bincount(minlength=5).cpu() - want).abs().max() <= 1


def test_no_rows(wq):
    assert wq.sample(torch.empty(0, 10, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


def test_captured_and_on_two_streams(wq):
    logits, draws, g = logits_of(4, 30000, BF16, seed=9)
    options = {"temperature": torch.full((4,), 0.8, device="cuda"), "top_k": 40, "top_p": 0.95}
    wq.sample(logits, draws, **options)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = wq.sample(logits, draws, **options)
    for seed in range(4):
        a, b, _ = logits_of(4, 30000, BF16, seed=20 + seed)
        logits.copy_(a), draws.copy_(b)
        options["temperature"].fill_(0.5 + 0.2 * seed)
        graph.replay()
        assert torch.equal(tokens.cpu(), defined(a, b, **options))
        assert torch.equal(tokens, wq.sample(logits, draws, **options))
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [logits_of(64, 20000, FP32, seed=30 + i) for i in range(2)]
    torch.cuda.synchronize()
    found = []
    for stream, (l, u, _) in zip(streams, inputs):
        with torch.cuda.stream(stream):
            found.append(wq.sample(l, u, top_k=50, top_p=0.9))
    torch.cuda.synchronize()
    for tokens, (l, u, _) in zip(found, inputs):
        assert torch.equal(tokens.cpu(), defined(l, u, top_k=50, top_p=0.9))


@pytest.mark.parametrize("vocabulary", [1500, 9000, 20000])
def test_lists_in_lds_in_memory_and_too_long(wq, vocabulary):
    """All of a row's logits in two or three bins: lists of keys of up to 2048, up to 16384, and rows that are read again."""
    g = torch.Generator(device="cuda").manual_seed(vocabulary)
    logits = torch.rand(5, vocabulary, generator=g, device="cuda") * 0.05
    draws = torch.rand(5, generator=g, device="cuda")
    for dtype in (FP32, BF16, FP16):
        l = logits.to(dtype)
        for options in ({"top_k": vocabulary // 3}, {"top_k": 700, "top_p": 0.4}, {"top_p": 0.6}, {"top_k": vocabulary // 2, "top_p": 0.5, "min_p": 0.97}, {"top_k": 1000}):
            assert torch.equal(wq.sample(l, draws, **options).cpu(), defined(l, draws, **options)), (dtype, options)


def test_large_vocabulary(wq):
    """3000001 tokens: weights in parts of 2^-40 (62 bits less 22 of an index), parts of several pieces. A part off by 2^-40 - 2^-44 moves the
    token only where a draw falls so near a border: with this seed it does not."""
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(2, 3_000_001, generator=g, device="cuda") * 3
    draws = torch.rand(2, generator=g, device="cuda")
    for options in ({}, {"top_k": 50}, {"top_p": 0.4}, {"top_k": 20000, "top_p": 0.9}, {"temperature": 0.0}):
        assert torch.equal(wq.sample(logits, draws, **options).cpu(), defined(logits, draws, **options)), options


@pytest.mark.parametrize("dtype", [FP16, FP32])
@pytest.mark.parametrize("options", [{}, {"top_k": 2000}, {"top_k": 4999}, {"top_k": 1025, "top_p": 0.6}, {"top_k": 3000, "min_p": 0.5}, {"top_k": 1000}, {"top_p": 0.5},
                                     {"top_k": 2000, "temperature": math.inf}])
def test_infinite_logits_share_all_weight(wq, dtype, options):
    """One to all of a row's logits infinite, beside finite ones and NaN: as many as, fewer and more than top-k, options as numbers and as tensors."""
    counts = [1, 2, 3, 10, 100, 1024, 1025, 1999, 2000, 2001, 4999, 5000]
    logits, _, g = logits_of(len(counts), 5000, dtype, seed=11)
    logits[::3, 5::7] = math.nan
    for row, count in enumerate(counts):
        logits[row, torch.randperm(5000, generator=g, device="cuda")[:count]] = math.inf
    for draws in (torch.linspace(0, 0.999, len(counts), device="cuda"), torch.linspace(1 - 2.0 ** -24, 0.1, len(counts), device="cuda")):
        want = defined(logits, draws, **options)
        assert torch.equal(wq.sample(logits, draws, **options).cpu(), want)
        tensors = {name: torch.full((len(counts),), value, dtype=torch.int32 if name == "top_k" else FP32, device="cuda") for name, value in options.items()}
        assert torch.equal(wq.sample(logits, draws, **tensors).cpu(), want)
        assert logits.cpu()[torch.arange(len(counts)), want].isinf().all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("temperature", [1e37, 5e37, 1e38, 3.4e38, math.inf])
def test_logits_whose_differences_pass_fp32(wq, dtype, temperature):
    """Logits over all of the type's range under temperatures alike: the largest one's distance to others is beyond FP32, their weights are not 0."""
    most = torch.finfo(dtype).max
    g = torch.Generator(device="cuda").manual_seed(12)
    logits = ((2 * torch.rand(6, 4000, generator=g, device="cuda", dtype=torch.float64) - 1) * most).to(dtype)
    logits[0, 17], logits[1, 3000], logits[2, 5] = most, most, -most
    draws = torch.rand(6, generator=g, device="cuda")
    for options in ({}, {"top_k": 40}, {"top_k": 3900}, {"top_p": 0.95}, {"top_p": 0.999, "top_k": 3990}, {"min_p": 0.01}):
        assert torch.equal(wq.sample(logits, draws, temperature=temperature, **options).cpu(), defined(logits, draws, temperature=temperature, **options)), options
    two = torch.tensor([[most, -most]], dtype=dtype, device="cuda")
    for options in ({}, {"top_k": 1}, {"top_p": 0.9999}):
        late = torch.tensor([1 - 2.0 ** -24], device="cuda")
        assert torch.equal(wq.sample(two, late, temperature=temperature, **options).cpu(), defined(two, late, temperature=temperature, **options)), options


@pytest.mark.parametrize("vocabulary,above", [(131072, 28.0), (2 ** 18, 27.0), (2 ** 18 + 1, 28.0), (2 ** 20, 28.0), (3_000_001, 30.0), (2 ** 24, 28.0), (2 ** 24, 31.0), (2 ** 24, 2.0)])
def test_a_peak_over_a_flat_tail(wq, vocabulary, above):
    """One logit `above` all others, which are alike, against the weights themselves (the peak's 1, the others' exp(-above), not rounded): the running weights
    beside the token drawn enclose the draw's. Every weight is rounded by half a unit, 2^-45 of the heaviest up to 2^18 tokens; above, 2^-53, or less than
    2^-62 of the sum (units of 2^(ceil(log2 sum) - 62)): 2^-27 of the sum for all tokens of a row. The kept sum of a top-p is the
    border's, off by as much again and a token."""
    w, peak = math.exp(-above), vocabulary // 3
    row = torch.zeros(1, vocabulary, device="cuda")
    row[0, peak] = above
    draws = torch.tensor([0.0, 0.5, 1 - 1000 * 2.0 ** -24, 1 - 200 * 2.0 ** -24, 1 - 100 * 2.0 ** -24, 1 - 30 * 2.0 ** -24, 1 - 2.0 ** -23, 1 - 2.0 ** -24], device="cuda")
    n = len(draws)
    weigh = lambda count: max(0.0, count) * w  # of that many tokens of the tail
    upto = lambda t: weigh(t + 1 if t < peak else t) + (1.0 if t >= peak else 0.0)  # the running weight with token t
    total = upto(vocabulary - 1)
    bound = 2.0 ** -27 * total
    for options, kept, slack in (({}, total, 0.0), ({"min_p": 0.9 * w}, total, 0.0), ({"top_k": vocabulary - 1}, total - w, 0.0),
                                 ({"top_p": 1 - 2.0 ** -24}, total * (1 - 2.0 ** -24), w + bound)):
        tokens = wq.sample(row.expand(n, vocabulary), draws, **options).tolist()
        for u, t in zip(draws.tolist(), tokens):
            assert upto(t - 1) - bound - slack <= u * kept <= upto(t) + bound + slack, (options, u, t)
        assert tokens == sorted(tokens)


def test_rows_of_all_kinds_over_a_large_vocabulary(wq):
    """Above 2^18 tokens weights have a unit of their own in every row: equal logits, one above all, infinities, NaN, greedy rows and masked ones side by side."""
    vocabulary = 2 ** 18 + 5
    logits, draws, _ = logits_of(9, vocabulary, FP32, seed=13)
    logits[0] = 2.5
    logits[1, 77] = 1000.0
    logits[2, 1000::5] = math.inf
    logits[3, ::2] = math.nan
    logits[4] = -math.inf
    logits[5, 200000:] = -math.inf
    logits[6] = math.nan
    temperature = torch.tensor([1.0, 1.0, 0.7, 1.3, 1.0, 0.5, 1.0, 0.0, 1e30], device="cuda")
    for options in ({}, {"top_k": 100000}, {"top_k": 30}, {"top_p": 0.7}, {"top_k": 5000, "top_p": 0.9, "min_p": 1e-4}):
        assert torch.equal(wq.sample(logits, draws, temperature=temperature, **options).cpu(), defined(logits, draws, temperature=temperature, **options)), options


@pytest.mark.parametrize("rows,vocabulary", [(9001, 9000), (16384, 9000), (2 ** 17, 300)])
@pytest.mark.parametrize("options", [{"top_k": 4000, "top_p": 0.7}, {"top_k": 700}, {"top_p": 0.9}, {"temperature": 0.0}])
def test_many_rows(wq, rows, vocabulary, options):
    """The most rows, and so many that lists of keys are shorter than a row's own: one flat row for all draws, of which every key lies in the cuts' bins."""
    print(f"rows {rows} {vocabulary} {options}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    row = torch.rand(1, vocabulary, generator=g, device="cuda") * 0.01
    draws = torch.rand(rows, generator=g, device="cuda")
    tokens = wq.sample(row.expand(rows, vocabulary), draws, **options).cpu()
    order = torch.sort(row[0].cpu(), descending=True, stable=True).indices
    if options.get("temperature") == 0.0:
        assert (tokens == order[0]).all()
        return
    weight = torch.round(torch.exp((row[0] - row.max()).cpu().double()) * 2.0 ** 44).long()
    kept = weight[order]
    kept[min(options.get("top_k", vocabulary), vocabulary):] = 0
    mass = torch.cumsum(kept, 0)
    if "top_p" in options:
        kept[mass - kept >= math.ceil(Fraction(torch.tensor(options["top_p"]).item()) * mass[-1].item())] = 0
    left = torch.zeros_like(weight)
    left[order] = kept
    upto = torch.cumsum(left, 0)
    total = upto[-1].item()
    targets = torch.tensor([math.floor(Fraction(u) * total) for u in draws.tolist()])
    assert torch.equal(tokens, torch.searchsorted(upto, targets, right=True))


def test_memory_of_a_call(wq):
    """1024 rows over 300 tokens: 15 KB a row and 8 bytes a token, with nothing cut the first only."""
    logits, draws, _ = logits_of(1024, 300, BF16, seed=14)
    for options, most in (({"top_k": 40}, 1024 * (16384 + 8 * 300)), ({"top_p": torch.full((1024,), 0.9, device="cuda")}, 1024 * (16384 + 8 * 300)), ({}, 1024 * 16384),
                          ({"temperature": 0.0, "top_k": 300}, 1024 * 16384)):
        want = defined(logits[:64], draws[:64], **{name: option[:64] if isinstance(option, torch.Tensor) else option for name, option in options.items()})
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        tokens = wq.sample(logits, draws, **options)
        assert torch.cuda.max_memory_allocated() - before <= most + 1024 * 8 + 2 ** 20
        assert torch.equal(tokens[:64].cpu(), want)
