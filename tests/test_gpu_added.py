"""add_prepare() and Prepared.values() on the GPU: bit for bit against the FP32 sum and prepare() of it, and against 64 bits.

Tolerance of a value against 64 bits: half a step of its scale (a code; a 254th of that with a remainder) and half a step of the 16-bit output,
besides the FP32 arithmetic before the code. That is, relative to the row's largest value: the squares' sum is off by one rounding a
chain's link (K / 256 of them and 8 more over the lanes, K <= 16384: at most 72) and its root by half as much, the division, the root, the two
products and the quotient by 8 more; ConvRot's stages add at most 4 of 6 operations each on values up to 2 x 4 stages larger, 2^8 in
all: (72 / 2 + 8 + 24) 2^-24 < 2^-17, and 2^-9 with a rotation."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def inputs(m, k, dtype, seed=0, scaled=True, pitch=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = lambda: torch.randn(m, k + pitch, generator=g, device="cuda").to(dtype)[:, :k]
    x, residual = rows(), rows()
    residual[:, torch.randperm(k, generator=g, device="cuda")[:3]] *= 30
    scale = torch.randn(k, generator=g, device="cuda").to(dtype) if scaled else None
    weight = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).to(dtype)
    return x, residual, scale, weight


def summed(x, residual, scale):
    """residual + scale * x with one rounding to FP32, one to the type (a product of 16-bit values is exact in FP32 but for the sum's rounding)."""
    branch = x.double() if scale is None else x.double() * scale.double()
    return (residual.double() + branch).float().to(x.dtype)


def same(a, b):
    return torch.equal(a.view(torch.int16) if a.dtype in (BF16, FP16) else a, b.view(torch.int16) if b.dtype in (BF16, FP16) else b)


def check(wq, prepared, total, x, residual, scale, weight, path, group, eps=1e-6):
    want = summed(x, residual, scale)
    assert same(total, want)
    other = wq.prepare(want, group, path, "rms_norm", weight, eps)
    assert prepared.path == path and prepared.dtype == x.dtype
    assert same(prepared.x, other.x)
    for a, b in ((prepared.lo, other.lo), (prepared.scale, other.scale)):
        assert (a is None) == (b is None) and (a is None or same(a, b))


@pytest.mark.parametrize("path", ["block", "exact", "row", "small"])
@pytest.mark.parametrize("m,k,dtype,group", [(1, 8, BF16, 0), (1, 5120, BF16, 0), (2, 2048, FP16, 256), (3, 2056, BF16, 0), (5, 4104, FP16, 0), (33, 1536, BF16, 64),
                                             (7, 7168, FP16, 16), (2, 8200, BF16, 0), (300, 4096, BF16, 256), (300, 5120, FP16, 0), (260, 6152, BF16, 0),
                                             (400, 1000, FP16, 0), (270, 13824, BF16, 0), (3, 16384, FP16, 256), (3, 16392, BF16, 0), (2, 20480, FP16, 64)])
def test_same_bits_as_prepare_of_the_sum(wq, path, m, k, dtype, group):
    print(f"added {path} {m} {k} {dtype} {group}", flush=True)
    x, residual, scale, weight = inputs(m, k, dtype, seed=m + k, scaled=m % 2 == 1)
    prepared, total = wq.add_prepare(x, residual, scale, group=group, path=path, act_weight=weight, eps=1e-6)
    check(wq, prepared, total, x, residual, scale, weight, path, group)


@pytest.mark.parametrize("path", ["block", "exact", "row", "lines"])
@pytest.mark.parametrize("m,k", [(1, 5120), (40, 2048), (300, 4104), (2, 20480)])
@pytest.mark.parametrize("over", ["residual", "x", "apart"])
def test_written_in_place_and_with_pitches(wq, path, m, k, over):
    print(f"in place {path} {m} {k} {over}", flush=True)
    x, residual, scale, weight = inputs(m, k, BF16, seed=m, pitch=16)
    before = x.clone(), residual.clone()
    out = residual if over == "residual" else x if over == "x" else torch.zeros(m, k + 8, dtype=BF16, device="cuda")[:, :k]
    prepared, total = wq.add_prepare(x, residual, scale, path=path, act_weight=weight, eps=1e-6, out=out)
    assert total is out
    check(wq, prepared, total, *before, scale, weight, path, 0)
    if over != "x":
        assert same(x, before[0])
    if over != "residual":
        assert same(residual, before[1])


def test_neighbouring_rows_of_one_buffer(wq):
    """[branch | residual | sum] side by side in rows of one tensor: they interleave and do not overlap."""
    m, k = 9, 512
    held = torch.randn(m, 3 * k, device="cuda").to(FP16)
    x, residual, out = held.split(k, 1)
    a, b = x.clone(), residual.clone()
    prepared, total = wq.add_prepare(x, residual, path="row", out=out)
    check(wq, prepared, total, a, b, None, None, "row", 0, 0.0)
    assert same(x, a) and same(residual, b)


@pytest.mark.parametrize("path", ["block", "exact", "row"])
@pytest.mark.parametrize("m,k,group", [(1, 40, 0), (4, 2048, 256), (65, 4104, 0), (3, 8192, 16)])
def test_values_against_64_bits(wq, path, m, k, group):
    print(f"values {path} {m} {k} {group}", flush=True)
    x, residual, scale, weight = inputs(m, k, FP16, seed=k)
    prepared, total = wq.add_prepare(x, residual, scale, group=group, path=path, act_weight=weight, eps=1e-6)
    v = total.double()
    v = v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * weight.double()
    if group:
        step = (1 - 2 * torch.eye(4, dtype=torch.float64).flip(0)) / 2
        turn = step
        while len(turn) < group:
            turn = torch.kron(step, turn)
        v = (v.reshape(-1, group) @ turn.cuda()).reshape(m, k)
    size = 128 if path == "block" else k
    top = torch.cat([p.abs().amax(1, keepdim=True).expand_as(p) for p in v.split(size, 1)], 1)
    row = v.abs().amax(1, keepdim=True)
    limit = top / 127 / 2 / (254 if path == "exact" else 1) * (1 + 2 ** -10) + row * (2.0 ** -9 if group else 2.0 ** -17) + v.abs() * 2.0 ** -11 + 2.0 ** -25
    values = prepared.values()
    assert values.dtype == FP16
    assert ((values.double() - v).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("path", ["block", "exact", "row", "lines"])
def test_values_of_prepare(wq, dtype, path):
    """Codes of prepare(): the FP64 product of code and scale, off by two FP32 roundings (and 254's inverse, rounded: 2^-24 of a part of
    at most half a step) and the output's."""
    x = torch.randn(11, 776, device="cuda").to(dtype)
    if path == "lines":
        if dtype != torch.float32:
            assert wq.prepare(x, path=path).values() is x
        return
    p = wq.prepare(x, path=path)
    code = p.x.double() + (0.0 if p.lo is None else p.lo.double() / 254)
    scale = p.scale.double().repeat_interleave(128, 1)[:, :776] if path == "block" else p.scale.double()[:, None]
    want = code * scale
    half = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    assert ((p.values().double() - want).abs() <= want.abs() * (half * 1.001 + 2.0 ** -23) + 2.0 ** -25).all()
    part = p.rows(3, 7)
    assert same(part.values(), p.values()[3:7])


def test_zeros_infinities_and_nan_stay_in_their_rows(wq):
    for path in ("block", "exact", "row", "small"):
        x, residual, _, weight = inputs(6, 1024, BF16, scaled=False)
        clean = wq.add_prepare(x, residual, path=path, act_weight=weight, eps=1e-6)
        x[1, 5], residual[2, 7], x[4] = float("nan"), float("inf"), 0
        residual[4] = 0
        prepared, total = wq.add_prepare(x, residual, path=path, act_weight=weight, eps=1e-6)
        check(wq, prepared, total, x, residual, None, weight, path, 0) if path == "small" else None
        assert total[1, 5].isnan() and total[2, 7].isinf() and not total[4].any()
        assert not prepared.values()[4].any()
        for row in (0, 3, 5):
            assert same(prepared.values()[row], clean[0].values()[row])


def test_no_rows(wq):
    for path in ("block", "exact", "row", "small"):
        x = torch.empty(0, 256, dtype=BF16, device="cuda")
        prepared, total = wq.add_prepare(x, x.clone(), path=path)
        assert total.shape == (0, 256) and prepared.values().shape == (0, 256)


def test_captured_and_on_another_stream(wq):
    x, residual, scale, weight = inputs(4, 5120, BF16)
    graph = torch.cuda.CUDAGraph()
    wq.add_prepare(x, residual, scale, path="exact", act_weight=weight, eps=1e-6)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        prepared, total = wq.add_prepare(x, residual, scale, path="exact", act_weight=weight, eps=1e-6)
    for seed in range(4):
        a, b, _, _ = inputs(4, 5120, BF16, seed=10 + seed)
        x.copy_(a), residual.copy_(b)
        graph.replay()
        check(wq, prepared, total, a, b, scale, weight, "exact", 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prepared, total = wq.add_prepare(x, residual, scale, path="block", act_weight=weight, eps=1e-6)
    torch.cuda.current_stream().wait_stream(side)
    check(wq, prepared, total, x, residual, scale, weight, "block", 0)


def test_into_linear_prepared(wq):
    x, residual, scale, weight = inputs(40, 1024, BF16)
    w = torch.randint(-127, 128, (384, 1024), dtype=torch.int8, device="cuda")
    s = torch.rand(384, device="cuda") / 127
    for path in ("block", "exact", "row"):
        prepared, total = wq.add_prepare(x, residual, scale, path=path, act_weight=weight, eps=1e-6)
        assert same(wq.linear_prepared(prepared, w, s), wq.linear(total, w, s, mode=path, act="rms_norm", act_weight=weight, eps=1e-6))


@pytest.mark.parametrize("path", ["block", "exact", "row", "small"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,group", [(7, 1024, 0), (7, 2056, 0), (7, 4096, 256), (7, 8200, 0), (600, 4104, 0), (7, 16392, 0)])
def test_rows_of_infinities_and_nan_as_prepare_has_them(wq, path, dtype, m, k, group):
    """Codes, remainders and scales of rows with NaN, one or two infinities, or nothing but zeros are prepare()'s of the sum too (NaN of any
    payload alike)."""
    print(f"not finite {path} {dtype} {m} {k} {group}", flush=True)
    x, residual, scale, weight = inputs(m, k, dtype, seed=k)
    x[1, 5], residual[2, k - 1] = float("nan"), float("inf")
    residual[3, 0], residual[3, k // 2] = float("inf"), float("-inf")
    x[4] = residual[4] = 0
    residual[5] = float("nan")
    residual[6] = torch.finfo(dtype).max
    prepared, total = wq.add_prepare(x, residual, scale, group=group, path=path, act_weight=weight, eps=1e-6)
    other = wq.prepare(total, group, path, "rms_norm", weight, 1e-6)
    for a, b in ((prepared.x, other.x), (prepared.lo, other.lo), (prepared.scale, other.scale)):
        assert (a is None) == (b is None)
        if a is not None and a.is_floating_point():
            assert torch.equal(a.isnan(), b.isnan())
            a, b = (torch.where(t.isnan(), torch.zeros_like(t), t) for t in (a, b))
        assert a is None or same(a, b)
