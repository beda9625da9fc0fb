"""route() and experts() on the GPU against 64 bits.

Tolerances. A sum of n products in FP32, in any order, is off by at most n u times the sum of their magnitudes; u = 2^-23 leaves room for
matrix instructions that cut off instead of rounding. That bounds gate and up (n = K); silu's slope is at most 1.1, its FP32 value within 2^-21 of
itself; the hidden value is held within 2^-17; the second product's sum (n = 2 hidden + top, for the two parts of a hidden value) is bounded
likewise; scales and weights take one rounding each; the output one to its type. A route's weights are FP64 rounded once to FP32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def layer(g, count, k, hidden):
    codes = lambda *shape: torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    scales = lambda *shape: (0.5 + torch.rand(*shape, generator=g, device="cuda")) / 74 * (k if shape[-1] == 2 * hidden else hidden) ** -0.5
    return codes(count, 2 * hidden, k), scales(count, 2 * hidden), codes(count, k, hidden), scales(count, k)


def expected(x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual=None, residual_scale=None):
    """(the layer in 64 bits, how far the kernel's output may be from it)."""
    tokens, k = x.shape
    hidden, top = down.shape[2], ids.shape[1]
    out = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    off, size = torch.zeros_like(out), torch.zeros_like(out)
    u = 2.0 ** -23
    for t in range(tokens):
        for j in range(top):
            e = ids[t, j].item()
            if not 0 <= e < len(down):
                continue
            a, v = gate_up[e].double() * gate_up_scale[e].double()[:, None], x[t].double()
            both, wide = a @ v, a.abs() @ v.abs()
            gate, up = both[:hidden], both[hidden:]
            d_gate, d_up = (wide * (k + 2) * u).split(hidden)
            silu = gate * torch.sigmoid(gate)
            h = silu * up
            d_h = 1.1 * d_gate * (up.abs() + d_up) + silu.abs() * d_up + h.abs() * (2.0 ** -21 + 2.0 ** -17) + 2.0 ** -126
            b, w = down[e].double() * down_scale[e].double()[:, None], weights[t, j].double()
            out[t] += w * (b @ h)
            reach = w.abs() * (b.abs() @ (h.abs() + d_h))
            size[t] += reach
            off[t] += w.abs() * (b.abs() @ d_h) + reach * (2 * hidden + 4) * u
    off += size * top * u
    if residual is not None:
        scale = 1.0 if residual_scale is None else residual_scale.double()
        out, off = residual.double() + scale * out, off * (1.0 if residual_scale is None else scale.abs())
    half = 2.0 ** -8 if x.dtype == BF16 else 2.0 ** -11
    return out, off + (out.abs() + off) * (half + u) + (2.0 ** -25 if x.dtype == FP16 else 2.0 ** -134)


def check(wq, x, ids, weights, parts, residual=None, residual_scale=None, out=None):
    want, off = expected(x, ids, weights, *parts, residual=residual, residual_scale=residual_scale)
    y = wq.experts(x, (ids, weights), *parts, residual=residual, residual_scale=residual_scale, out=out)
    assert y.dtype == x.dtype and y.shape == x.shape
    # from half a step past the type's largest value on, the nearest value is an infinity (FP16: 65504 + 16)
    most = torch.finfo(x.dtype).max
    beyond = want.abs() - off >= most * (1 + torch.finfo(x.dtype).eps / 2)
    near = (want.abs() + off >= most) & ~beyond & y.isinf()
    bad = torch.where(beyond, y.double() != want.sign() * float("inf"), ((y.double() - want).abs() > off) & ~near)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((y.double() - want).abs() / off).max().item():.3g} of the tolerance"
    return y


def choices(g, tokens, top, count):
    ids = torch.stack([torch.randperm(count, generator=g, device="cuda")[:top] for _ in range(tokens)]).int()
    return ids, torch.rand(tokens, top, generator=g, device="cuda") + 0.1


@pytest.mark.parametrize("tokens,k,hidden,count,top,dtype", [
    (1, 16, 16, 1, 1, BF16), (1, 2048, 1024, 64, 8, BF16), (1, 2048, 768, 9, 8, FP16), (2, 512, 256, 16, 4, BF16), (3, 1552, 592, 21, 3, FP16),
    (4, 1040, 80, 8, 8, BF16), (5, 272, 48, 5, 5, FP16), (7, 5120, 144, 3, 2, BF16), (8, 256, 2064, 8, 2, FP16), (13, 1296, 320, 6, 2, BF16),
    (16, 1024, 512, 128, 8, BF16), (33, 528, 208, 64, 6, FP16), (40, 384, 96, 2, 2, BF16), (70, 144, 112, 4, 3, FP16)])
def test_against_64_bits(wq, tokens, k, hidden, count, top, dtype):
    print(f"experts {tokens} {k} {hidden} {count} {top} {dtype}", flush=True)
    g = generator(tokens * 7 + k)
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    ids, weights = choices(g, tokens, top, count)
    residual = torch.randn(tokens, k, generator=g, device="cuda").to(dtype) if tokens % 2 else None
    scale = torch.randn(k, generator=g, device="cuda").to(dtype) if tokens % 4 == 1 else None
    check(wq, x, ids, weights, layer(g, count, k, hidden), residual, scale)


@pytest.mark.parametrize("counts", [(1, 4, 5, 0), (8, 9, 2, 16), (17, 32, 3, 1), (33, 64, 4, 8), (65, 129, 0, 12), (4, 4, 4, 4)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_any_number_of_tokens_an_expert(wq, counts, dtype):
    """One choice a token: `counts` of them for each expert, in a mixed order."""
    print(f"counts {counts} {dtype}", flush=True)
    g = generator(sum(counts))
    ids = torch.cat([torch.full((n,), e, device="cuda") for e, n in enumerate(counts)]).int()
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")][:, None].contiguous()
    x = torch.randn(len(ids), 336, generator=g, device="cuda").to(dtype)
    check(wq, x, ids, torch.rand(len(ids), 1, generator=g, device="cuda"), layer(g, len(counts), 336, 176))


@pytest.mark.parametrize("tokens,k,hidden,count,top,dtype", [
    (1, 256, 2064, 70, 65, BF16), (1, 512, 1552, 20, 17, FP16), (1, 4096, 48, 64, 64, BF16), (2, 2048, 528, 64, 8, FP16), (4, 4112, 272, 16, 4, BF16), (6, 304, 1040, 96, 12, BF16)])
def test_forms_of_few_tokens(wq, tokens, k, hidden, count, top, dtype):
    """One token of many choices and long rows; two to six around the borders between shared tiles and shared tokens."""
    print(f"few {tokens} {k} {hidden} {count} {top} {dtype}", flush=True)
    g = generator(k + hidden)
    x, residual = (torch.randn(tokens, k, generator=g, device="cuda").to(dtype) for _ in range(2))
    ids, weights = choices(g, tokens, top, count)
    ids[0, top // 2] = -1
    check(wq, x, ids, weights, layer(g, count, k, hidden), residual)


def test_all_of_many_tokens_on_one_expert(wq):
    g = generator(12)
    parts = layer(g, 3, 128, 48)
    x = torch.randn(333, 128, generator=g, device="cuda").to(BF16)
    ids = torch.ones(333, 1, dtype=torch.int32, device="cuda")
    check(wq, x, ids, torch.rand(333, 1, generator=g, device="cuda"), parts)
    twice = torch.ones(8, 2, dtype=torch.int32, device="cuda")  # 16 choices of 8 tokens
    check(wq, x[:8], twice, torch.rand(8, 2, generator=g, device="cuda"), parts)


def test_experts_outside_and_twice(wq):
    g = generator(3)
    parts = layer(g, 6, 256, 64)
    x, residual = (torch.randn(5, 256, generator=g, device="cuda").to(BF16) for _ in range(2))
    big = 2 ** 31 - 1
    ids = torch.tensor([[-1, 2, 6], [3, 3, 3], [-1, -5, big], [5, 0, 5], [6, 7, 1]], dtype=torch.int32, device="cuda")
    weights = torch.rand(5, 3, generator=g, device="cuda")
    y = check(wq, x, ids, weights, parts)
    assert not y[2].any()
    y = check(wq, x, ids, weights, parts, residual)
    assert torch.equal(y[2], residual[2])
    one = torch.full((1, 1), 9, dtype=torch.int32, device="cuda")
    assert not wq.experts(x[:1], (one, weights[:1, :1].contiguous()), *parts).any()


def test_most_choices_and_none(wq):
    g = generator(4)
    parts = layer(g, 3, 64, 32)
    x = torch.randn(2048, 64, generator=g, device="cuda").to(FP16)
    ids = torch.randint(0, 3, (2048, 2), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(2048, 2, generator=g, device="cuda")
    y = wq.experts(x, (ids, weights), *parts)
    for at in (0, 1000, 2040):  # the same rows in small calls: every token's sums are its own
        few = slice(at, at + 8)
        want, off = expected(x[few], ids[few], weights[few], *parts)
        assert ((y[few].double() - want).abs() <= off).all()
    with pytest.raises(ValueError):
        wq.experts(torch.cat([x, x[:1]]), (torch.cat([ids, ids[:1]]), torch.cat([weights, weights[:1]])), *parts)
    assert wq.experts(x[:0], (ids[:0], weights[:0]), *parts).shape == (0, 64)


def test_rows_apart_and_in_place(wq):
    g = generator(5)
    parts = layer(g, 7, 320, 96)
    held = torch.randn(6, 3 * 320, generator=g, device="cuda").to(BF16)
    x, residual, out = held.split(320, 1)
    ids, weights = choices(g, 6, 3, 7)
    before = held.clone()
    y = check(wq, x, ids, weights, parts, residual, out=out)
    assert y.data_ptr() == out.data_ptr() and torch.equal(held[:, :640], before[:, :640])
    want = out.clone()
    assert torch.equal(wq.experts(x, (ids, weights), *parts, residual=residual, out=residual), want)
    residual.copy_(before[:, 320:640])
    assert torch.equal(wq.experts(x, (ids, weights), *parts, residual=residual, out=x), want)


def test_infinities_and_nan_stay_in_their_rows(wq):
    g = generator(6)
    parts = layer(g, 4, 256, 64)
    x = torch.randn(12, 256, generator=g, device="cuda").to(BF16)
    ids, weights = choices(g, 12, 2, 4)
    clean = wq.experts(x, (ids, weights), *parts)
    x[3, 7], x[9, 0] = float("nan"), float("inf")
    y = wq.experts(x, (ids, weights), *parts)
    assert y[3].isnan().all()
    keep = [t for t in range(12) if t not in (3, 9)]
    assert torch.equal(y[keep], clean[keep])


def test_large_hidden_values(wq):
    """Products past FP16's range: the hidden values are not cut off at 65504."""
    g = generator(7)
    parts = list(layer(g, 2, 128, 64))
    parts[1] = parts[1] * 300
    parts[3] = parts[3] / 1000
    x = (torch.randn(3, 128, generator=g, device="cuda") * 30).to(FP16)
    ids, weights = choices(g, 3, 2, 2)
    y = check(wq, x, ids, weights, parts)
    e = ids[0, 0].item()
    gate, up = ((parts[0][e].double() * parts[1][e].double()[:, None]) @ x[0].double()).chunk(2)
    assert (gate * torch.sigmoid(gate) * up).abs().max() > 65504 and y.isfinite().sum() > y.numel() / 2


def test_weights_past_32_bit_offsets(wq):
    count, k, hidden = 66, 8192, 4096
    free = torch.cuda.mem_get_info()[0]
    assert free > 12 << 30
    g = generator(8)
    small = layer(g, 1, k, hidden)
    large = [torch.zeros(count, *t.shape[1:], dtype=t.dtype, device="cuda") for t in small]
    for a, b in zip(large, small):
        a[count - 1] = b[0]
    x = torch.randn(2, k, generator=g, device="cuda").to(BF16)
    ids, weights = torch.full((2, 1), count - 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")
    assert large[0].numel() > 2 ** 32
    y = wq.experts(x, (ids, weights), *large)
    assert torch.equal(y, wq.experts(x, (torch.zeros_like(ids), weights), *small)) and y.any()


# ---- the router --------------------------------------------------------------------------------------------------------
def routed(x, router, top, score="softmax", bias=None, normalise=True, factor=1.0):
    logits = x.cpu().double() @ router.cpu().double().T
    scores = torch.softmax(logits, 1) if score == "softmax" else torch.sigmoid(logits)
    wanted = scores if bias is None else scores + bias.cpu().double()
    ids = torch.sort(wanted, dim=1, descending=True, stable=True).indices[:, :top]
    weights = scores.gather(1, ids)
    return ids.int(), (weights / weights.sum(1, keepdim=True) if normalise else weights) * factor


@pytest.mark.parametrize("tokens,k,count,top,dtype,router_dtype", [(1, 8, 1, 1, BF16, BF16), (1, 2048, 64, 8, BF16, BF16), (3, 5120, 128, 8, FP16, FP32),
                                                                   (17, 1032, 160, 6, BF16, FP32), (16, 40, 65, 64, FP16, FP16), (5, 512, 1000, 10, FP32, FP32),
                                                                   (1000, 264, 8, 2, BF16, FP16), (33, 776, 257, 1, FP32, BF16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route(wq, tokens, k, count, top, dtype, router_dtype, score, biased):
    print(f"route {tokens} {k} {count} {top} {dtype} {router_dtype} {score} {biased}", flush=True)
    g = generator(tokens + k)
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    router = (torch.randn(count, k, generator=g, device="cuda") * 2 * k ** -0.5).to(router_dtype)
    bias = 0.1 * torch.randn(count, generator=g, device="cuda") if biased else None
    for normalise, factor in ((True, 1.0), (False, 2.5)):
        ids, weights = wq.route(x, router, top, score=score, bias=bias, normalise=normalise, factor=factor)
        want_ids, want = routed(x, router, top, score, bias, normalise, factor)
        assert torch.equal(ids.cpu(), want_ids)
        # FP64 sums and functions, one rounding to FP32
        assert ((weights.cpu().double() - want).abs() <= want * (2.0 ** -24 + 2.0 ** -40)).all()


def test_route_ties_go_to_the_lowest_index(wq):
    g = generator(9)
    router = torch.randn(4, 64, generator=g, device="cuda").to(BF16).repeat(33, 1)  # 132 experts, each 33 times
    x = torch.randn(6, 64, generator=g, device="cuda").to(BF16)
    for top in (1, 5, 40):
        ids, weights = wq.route(x, router, top)
        want, _ = routed(x, router, top)
        assert torch.equal(ids.cpu(), want)
    ids, weights = wq.route(torch.zeros_like(x), router, 7)
    assert torch.equal(ids.cpu(), torch.arange(7).int().expand(6, 7)) and torch.equal(weights, torch.full_like(weights, 1 / 7))


def test_route_of_nan_rows(wq):
    g = generator(10)
    x, router = torch.randn(5, 64, generator=g, device="cuda").to(BF16), torch.randn(40, 64, generator=g, device="cuda").to(BF16)
    x[2, 3] = float("nan")
    clean = [0, 1, 3, 4]
    for score in ("softmax", "sigmoid"):
        ids, weights = wq.route(x, router, 4, score=score)
        assert torch.equal(ids[2].cpu(), torch.arange(4).int()) and weights[2].isnan().all()
        want, _ = routed(x[clean], router, 4, score)
        assert torch.equal(ids[clean].cpu(), want)
    router[7] = float("nan")  # one expert's: the others are chosen before it
    ids, _ = wq.route(x[:2], router, 40, score="sigmoid")
    assert (ids[:, -1] == 7).all() and all(sorted(row) == list(range(40)) for row in ids.tolist())


def test_whole_layer_captured(wq):
    g = generator(11)
    parts = layer(g, 16, 512, 128)
    router = torch.randn(16, 512, generator=g, device="cuda").to(BF16)
    x, residual = (torch.randn(3, 512, generator=g, device="cuda").to(BF16) for _ in range(2))

    def step():
        return wq.experts(x, wq.route(x, router, 4), *parts, residual=residual)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for _ in range(4):
        x.copy_(torch.randn(3, 512, generator=g, device="cuda"))
        graph.replay()
        got = y.clone()
        assert torch.equal(got, step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)


def test_most_tokens_of_a_route(wq):
    """As many tokens as a route takes: rows at both ends and between them against the definition, all of them one expert each or more."""
    tokens = 65535 * 16
    g = generator(13)
    x = torch.randn(tokens, 16, generator=g, device="cuda").to(BF16)
    router = torch.randn(20, 16, generator=g, device="cuda").to(BF16)
    ids, weights = wq.route(x, router, 3)
    for at in (0, 1, 4000, 500_001, tokens - 33):
        want_ids, want = routed(x[at:at + 33], router, 3)
        assert torch.equal(ids[at:at + 33].cpu(), want_ids)
        assert ((weights[at:at + 33].cpu().double() - want).abs() <= want * (2.0 ** -24 + 2.0 ** -40)).all()
    assert ((ids >= 0) & (ids < 20)).all()
    with pytest.raises(ValueError):
        wq.route(torch.cat([x, x[:1]]), router, 3)
