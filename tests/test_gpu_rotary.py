"""Rotary positions on the GPU against 64 bits: styles, ladders, axes, types, odd token counts, strides, far and negative positions, part
of a head, in place, the inverse as gradient, a replayed graph.

Tolerance: half a step of the output type of the value, and for the angle's sine and cosine (within 2^-23: polynomials 2^-28, the
FP32 steps of their evaluation) and the two FP32 operations of a channel, 2^-22 (|a| + |b|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def exact(x, positions, sections, ladder, style, inverse=False, base=10000.0):
    pairs = sum(sections)
    steps = [i / n for n in sections for i in range(n)] if ladder == "axis" else [i / pairs for i in range(pairs)]
    frequency = torch.tensor([base ** -s for s in steps], dtype=torch.float64)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    angle = positions.cpu().reshape(positions.shape[0], -1)[:, axis].double() * frequency
    cos, sin = angle.cos()[:, None], (-angle.sin() if inverse else angle.sin())[:, None]
    x = x.cpu().double()
    out, size = x.clone(), x.abs()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if style == "pairs" else (slice(0, pairs), slice(pairs, 2 * pairs))
    out[..., a], out[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    both = x[..., a].abs() + x[..., b].abs()
    size[..., :2 * pairs] = 0
    size[..., a], size[..., b] = both, both
    turned = torch.zeros(x.shape[-1], dtype=torch.bool)
    turned[:2 * pairs] = True
    return out, size * turned


def check(got, x, *how, **more):
    want, size = exact(x, *how, **more)
    off = (got.cpu().double() - want).abs()
    info = torch.finfo(got.dtype)
    half_step = info.eps / 2 * want.abs().clamp(min=info.smallest_normal)  # below the normal range steps stay as they are
    bound = half_step + 2.0 ** -22 * size
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("style", ["pairs", "halves"])
@pytest.mark.parametrize("ladder", ["axis", "joint"])
@pytest.mark.parametrize("tokens,heads,head_dim,sections,far", [(1, 1, 8, (4,), 10), (1, 40, 128, (16, 24, 24), 10 ** 6), (7, 3, 80, (20,), 5000),
                                                                (257, 5, 64, (12, 12), 100), (1031, 12, 128, (22, 21, 21), 2 ** 31 - 1),
                                                                (33, 2, 96, (7, 6, 6), 1000), (65, 9, 256, (64, 64), 10 ** 6)])
def test_rotary(wq, dtype, style, ladder, tokens, heads, head_dim, sections, far):
    print(f"rotary {dtype} {style} {ladder} {tokens} {heads} {head_dim} {sections} {far}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    row = torch.randn(tokens, heads + 2, head_dim, generator=g, device="cuda").to(dtype)  # one projection, two key heads
    q, k = row[:, :heads], row[:, heads:]
    positions = torch.randint(-far, far, (tokens, len(sections)), generator=g, device="cuda").int()
    plan = wq.rotary_plan(sections, ladder=ladder, style=style)
    before = row.clone()
    for inverse in (False, True):
        rq, rk = wq.rotary((q, k), positions, plan, inverse=inverse)
        check(rq, q, positions, sections, ladder, style, inverse=inverse)
        check(rk, k, positions, sections, ladder, style, inverse=inverse)
    assert torch.equal(row, before)
    wide = torch.stack([positions.long(), positions.long()], -1)[..., 0]  # int64, strided
    assert torch.equal(wq.rotary(q, wide, plan, inverse=True), rq)
    assert wq.rotary((q, k), positions, plan, out=(q, k))[0] is q  # in place
    check(q, before[:, :heads], positions, sections, ladder, style)
    check(k, before[:, heads:], positions, sections, ladder, style)


def test_no_tokens(wq):
    plan = wq.rotary_plan((4,))
    assert wq.rotary(torch.empty(0, 2, 16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), plan).shape == (0, 2, 16)


@pytest.mark.parametrize("style", ["pairs", "halves"])
def test_gradient(wq, style):
    """For a loss sum(w * rotary(x)) the gradient is the inverse rotation of w; against differences in 64 bits (the rotation is linear,
    so that they have no error of their own but that of the FP32 output: 2^-24 of its size, and twice 2^-22 for the angles)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(5, 2, 16, generator=g, device="cuda") for _ in range(2))
    positions = torch.randint(0, 900, (5,), generator=g, device="cuda").int()
    plan = wq.rotary_plan((7,), style=style)
    grad = wq.rotary(w, positions, plan, inverse=True).double()
    loss = lambda v: (w.double() * wq.rotary(v, positions, plan).double()).sum()
    for token, head, channel in [(0, 0, 0), (1, 1, 3), (4, 0, 13), (2, 1, 7), (3, 0, 14), (3, 1, 15)]:
        e = torch.zeros_like(x)
        e[token, head, channel] = 1.0
        slope = loss(x + e) - loss(x - e)
        size = w[token, head].abs().sum().item() * (x.abs().max().item() + 1)
        assert abs(slope.item() / 2 - grad[token, head, channel].item()) <= size * 2.0 ** -20
    back = wq.rotary(wq.rotary(x, positions, plan), positions, plan, inverse=True)
    assert (back - x).abs().max() <= 2.0 ** -20 * x.abs().max()


def test_nonfinite_stays_in_its_pair(wq):
    x = torch.ones(2, 1, 16, device="cuda")
    x[0, 0, 2], x[1, 0, 15] = math.nan, math.inf
    y = wq.rotary(x, torch.tensor([3, 4], dtype=torch.int32, device="cuda"), wq.rotary_plan((6,)))
    finite = torch.isfinite(y).cpu()
    want = torch.ones(2, 1, 16, dtype=torch.bool)
    want[0, 0, 2] = want[0, 0, 3] = want[1, 0, 15] = False
    assert torch.equal(finite, want)


def test_graph_and_side_stream(wq):
    plan = wq.rotary_plan((32, 32))
    x, positions = torch.randn(70, 6, 128, device="cuda").half(), torch.arange(140, device="cuda").reshape(70, 2).int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = wq.rotary(x, positions, plan)
    torch.cuda.current_stream().wait_stream(side)
    check(y, x, positions, (32, 32), "axis", "pairs")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = wq.rotary(x, positions, plan)
    for r in range(4):
        positions += 1000 * r
        want = wq.rotary(x, positions, plan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("style", ["pairs", "halves"])
def test_far_positions_in_64_bits(wq, dtype, style):
    """Positions up to 2^44: the angle, from integers, is off by |p| 2^-65 turns, 2^-18.3 at most, of |a| + |b|."""
    from fractions import Fraction
    frequencies = [1.0, 0.7071, 0.3, 10000.0 ** -0.3, 1e-5, 123.456]
    plan = wq.rotary_plan((2, 4), style=style, frequencies=frequencies)
    g = torch.Generator(device="cuda").manual_seed(7)
    positions = torch.randint(-(2 ** 44), 2 ** 44, (37, 2), generator=g, device="cuda")
    x = torch.randn(37, 3, 16, generator=g, device="cuda").to(dtype)
    # 2 pi to 80 digits
    two_pi = Fraction("6.2831853071795864769252867665590057683943387987502116419498891846156328125724180")
    turn = lambda p, f: (p * Fraction(f) / two_pi) % 1
    axis = [0] * 2 + [1] * 4
    angle = torch.tensor([[2 * math.pi * float(turn(row[a], f)) for a, f in zip(axis, frequencies)] for row in positions.tolist()], dtype=torch.float64)
    for inverse in (False, True):
        got = wq.rotary(x, positions, plan, inverse=inverse).cpu().double()
        want, size = x.cpu().double(), torch.zeros(37, 3, 16, dtype=torch.float64)
        a, b = (slice(0, 12, 2), slice(1, 12, 2)) if style == "pairs" else (slice(0, 6), slice(6, 12))
        u, v, cos, sin = want[..., a].clone(), want[..., b].clone(), angle.cos()[:, None], (-angle.sin() if inverse else angle.sin())[:, None]
        want[..., a], want[..., b] = u * cos - v * sin, u * sin + v * cos
        size[..., a] = size[..., b] = u.abs() + v.abs()
        far = 2 * math.pi * 2.0 ** -65 * positions.abs().max().item()
        info = torch.finfo(dtype)
        bound = info.eps / 2 * want.abs().clamp(min=info.smallest_normal) + (2.0 ** -22 + far) * size
        assert ((got - want).abs() <= bound).all()
