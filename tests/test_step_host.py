"""The operators around the linears of a decode step (add_prepare, route, experts, sample), without a GPU: what they refuse, before anything is launched."""
import pytest
import torch

from wgpkernels_amd import int8 as wq

BF16, FP16 = torch.bfloat16, torch.float16


def rows(m=4, k=256, dtype=BF16):
    return torch.zeros(m, k, dtype=dtype)


ADDED = {
    "dimensions": lambda: (rows()[0], rows()[0], {}),
    "type": lambda: (rows(dtype=torch.float32), rows(dtype=torch.float32), {}),
    "mixed types": lambda: (rows(), rows(dtype=FP16), {}),
    "double": lambda: (rows(dtype=torch.float64), rows(dtype=torch.float64), {}),
    "shapes": lambda: (rows(), rows(5), {}),
    "broadcast": lambda: (rows(), rows(1), {}),
    "width": lambda: (rows(k=252), rows(k=252), {}),
    "no channels": lambda: (rows(k=0), rows(k=0), {}),
    "columns": lambda: (torch.zeros(256, 4, dtype=BF16).t(), rows(), {}),
    "many rows": lambda: (rows(1, 8).expand(2 ** 24, 8), rows(1, 8).expand(2 ** 24, 8), {}),
    "pitch": lambda: (rows(k=260)[:, :256], rows(), {}),
    "path": lambda: (rows(), rows(), {"path": "fast"}),
    "group": lambda: (rows(), rows(), {"group": 32}),
    "group width": lambda: (rows(k=264), rows(k=264), {"group": 16}),
    "scale shape": lambda: (rows(), rows(), {"residual_scale": torch.zeros(128, dtype=BF16)}),
    "scale type": lambda: (rows(), rows(), {"residual_scale": torch.zeros(256)}),
    "weight shape": lambda: (rows(), rows(), {"act_weight": torch.zeros(1, 256, dtype=BF16)}),
    "weight stride": lambda: (rows(), rows(), {"act_weight": torch.zeros(512, dtype=BF16)[::2]}),
    "cpu": lambda: (rows(), rows(), {}),
}


@pytest.mark.parametrize("change", list(ADDED))
def test_add_prepare_refuses(change):
    x, residual, options = ADDED[change]()
    with pytest.raises(ValueError):
        wq.add_prepare(x, residual, **options)


def test_sums_over_their_inputs():
    from wgpkernels_amd.int8._added import _check_sum, _rows_meet
    held = torch.zeros(8, 768, dtype=BF16)
    x, residual, out = held.split(256, 1)
    assert not _rows_meet(out, x) and not _rows_meet(x, out) and _rows_meet(x, x)
    assert _rows_meet(held[:, 8:264], x) and _rows_meet(held[2:4, :256], held[3:5, :256]) and not _rows_meet(held[:2, :256], held[2:4, :256])
    flat = torch.zeros(2048, dtype=BF16)
    assert _rows_meet(flat[:496].view(2, 248), flat[8:504].view(2, 248)) and not _rows_meet(flat[:496].view(2, 248), flat[496:992].view(2, 248))
    assert _rows_meet(flat[:496].view(2, 248), flat[:1024].view(2, 512)[:, :248]) and not _rows_meet(held[:2, 512:], held[2:4, :256])
    for bad in (held[:, 8:264], held[1:5, :256], rows(5), rows(dtype=FP16), rows(1).expand(4, 256), torch.zeros(4, 260, dtype=BF16)[:, :256]):
        a, b = (held[:, :256], rows(8)) if bad.shape[0] == 8 else (held[:4, :256], rows())
        with pytest.raises(ValueError):
            _check_sum(bad, a, b)


def test_prepared_values_refuse():
    codes = torch.zeros(4, 256, dtype=torch.int8)
    for p in (wq.Prepared("block", codes, None, torch.zeros(4), BF16), wq.Prepared("row", codes, None, torch.zeros(5), BF16),
              wq.Prepared("row", codes[:, :250], None, torch.zeros(4), BF16), wq.Prepared("row", codes[:, :128], None, torch.zeros(4), BF16)):
        with pytest.raises(ValueError):
            p.values()


def layer(count=4, k=64, hidden=32):
    return {"gate_up": torch.zeros(count, 2 * hidden, k, dtype=torch.int8), "gate_up_scale": torch.zeros(count, 2 * hidden),
            "down": torch.zeros(count, k, hidden, dtype=torch.int8), "down_scale": torch.zeros(count, k)}


def routes(tokens=3, top=2):
    return torch.zeros(tokens, top, dtype=torch.int32), torch.zeros(tokens, top)


EXPERTS = {
    "type": {"x": rows(3, 64, torch.float32)},
    "width": {"x": rows(3, 80)},
    "pitch": {"x": rows(3, 68)[:, :64]},
    "columns": {"x": torch.zeros(64, 3, dtype=BF16).t()},
    "tokens": {"x": rows(4, 64)},
    "ids type": {"routes": (torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))},
    "weights type": {"routes": (torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=BF16))},
    "weights shape": {"routes": (torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 1))},
    "ids strides": {"routes": (torch.zeros(2, 3, dtype=torch.int32).t(), torch.zeros(3, 2))},
    "no choices": {"routes": routes(3, 0)},
    "many choices": {"x": rows(2049, 64), "routes": routes(2049, 2)},
    "gate_up type": {"gate_up": torch.zeros(4, 64, 64)},
    "gate_up strides": {"gate_up": torch.zeros(4, 64, 128, dtype=torch.int8)[..., :64]},
    "hidden": {"gate_up": torch.zeros(4, 48, 64, dtype=torch.int8), "gate_up_scale": torch.zeros(4, 48)},
    "channels": {"x": rows(3, 72), **layer(k=72)},
    "down shape": {"down": torch.zeros(4, 64, 16, dtype=torch.int8)},
    "down experts": {"down": torch.zeros(3, 64, 32, dtype=torch.int8), "down_scale": torch.zeros(3, 64)},
    "scales": {"down_scale": torch.zeros(4, 32)},
    "scale type": {"gate_up_scale": torch.zeros(4, 64, dtype=BF16)},
    "group scales": {"down_scale": torch.zeros(4, 64, 1)},
    "residual": {"residual": rows(3, 64, FP16)},
    "residual shape": {"residual": rows(1, 64)},
    "residual_scale alone": {"residual_scale": torch.zeros(64, dtype=BF16)},
    "residual_scale": {"residual": rows(3, 64), "residual_scale": torch.zeros(64)},
    "spans 2 GiB": {"x": torch.zeros(3, 32768, dtype=BF16), "gate_up": torch.zeros(1, 65536, 32768, dtype=torch.int8, device="meta"),
                    "gate_up_scale": torch.zeros(1, 65536, device="meta"), "down": torch.zeros(1, 32768, 32768, dtype=torch.int8, device="meta"),
                    "down_scale": torch.zeros(1, 32768, device="meta")},
    "cpu": {},
}


@pytest.mark.parametrize("change", list(EXPERTS))
def test_experts_refuse(change):
    with pytest.raises(ValueError):
        wq.experts(**{"x": rows(3, 64), "routes": routes(), **layer(), **EXPERTS[change]})


ROUTE = {
    "type": {"x": rows(3, 64, torch.float64)},
    "width": {"x": rows(3, 72)},
    "pitch": {"x": rows(3, 68)[:, :64]},
    "router type": {"router": torch.zeros(8, 64, dtype=torch.float64)},
    "router strides": {"router": torch.zeros(64, 8).t()},
    "channels": {"x": rows(3, 60), "router": torch.zeros(8, 60)},
    "no experts": {"router": torch.zeros(0, 64)},
    "many experts": {"router": torch.zeros(1025, 64)},
    "no choice": {"top": 0},
    "more than there are": {"top": 9},
    "many choices": {"top": 65, "router": torch.zeros(100, 64)},
    "score": {"score": "linear"},
    "bias type": {"bias": torch.zeros(8, dtype=BF16)},
    "bias shape": {"bias": torch.zeros(8, 1)},
    "cpu": {},
}


@pytest.mark.parametrize("change", list(ROUTE))
def test_route_refuses(change):
    with pytest.raises(ValueError):
        wq.route(**{"x": rows(3, 64), "router": torch.zeros(8, 64), "top": 2, **ROUTE[change]})


SAMPLE = {
    "dimensions": {"logits": torch.zeros(5)},
    "type": {"logits": torch.zeros(3, 5, dtype=torch.float64)},
    "columns": {"logits": torch.zeros(5, 3).t()},
    "no vocabulary": {"logits": torch.zeros(3, 0)},
    "wide": {"logits": torch.zeros(3, 1).expand(3, 2 ** 24 + 1)},
    "many rows": {"logits": torch.zeros(1, 5).expand(2 ** 17 + 1, 5), "draws": torch.zeros(2 ** 17 + 1)},
    "draws shape": {"draws": torch.zeros(3, 1)},
    "draws type": {"draws": torch.zeros(3, dtype=torch.float64)},
    "draws strides": {"draws": torch.zeros(6)[::2]},
    "temperature type": {"temperature": torch.ones(3, dtype=BF16)},
    "temperature shape": {"temperature": torch.ones(1)},
    "top_k type": {"top_k": torch.ones(3)},
    "top_p strides": {"top_p": torch.ones(6)[::2]},
    "min_p shape": {"min_p": torch.ones(4)},
    "cpu": {},
}


@pytest.mark.parametrize("change", list(SAMPLE))
def test_sample_refuses(change):
    with pytest.raises(ValueError):
        wq.sample(**{"logits": torch.zeros(3, 5), "draws": torch.zeros(3), **SAMPLE[change]})


def test_a_launch_has_its_device_current(monkeypatch):
    """call_on() makes the tensors' GPU the current one around a call, and only where it is not."""
    from wgpkernels_amd.int8 import _native
    seen, entered = [], []

    class Device:
        def __init__(self, index):
            entered.append(index)

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *_):
            seen.append("out")

    class Library:
        def call(self, name, *args):
            seen.append((name, args))

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    _native.call_on(Library(), 0, "a", 1)
    _native.call_on(Library(), 1, "b", 2)
    assert seen == [("a", (1,)), "in", ("b", (2,)), "out"] and entered == [1]


def test_most_values_of_top_k():
    """A top_k beyond the C interface's 32 bits is all of the vocabulary, not its low bits."""
    from wgpkernels_amd.int8 import _sample
    assert min(2 ** 32 + 3, _sample.MAX_VOCABULARY) == 2 ** 24 and _sample._pair(min(2 ** 32 + 3, _sample.MAX_VOCABULARY)) == (None, 2 ** 24)


def test_entry_points_reject_before_a_launch():
    """The C interface's own checks: codes without a GPU touched."""
    lib = wq.library()
    add = lambda m=4, k=64, dtype=1, path=0, group=0: lib.wq8_add_prepare(None, k, None, k, None, None, k, path, None, None, None, m, k, dtype, group, None, 0.0, None)
    assert add(m=0) == 0
    assert [add(dtype=2), add(path=3), add(group=32)] == [-1] * 3 and [add(k=60), add(k=0), add(m=-1), add(m=2 ** 24), add(k=24, group=16)] == [-2] * 5
    assert lib.wq8_prepared_values(None, None, None, None, 0, 64, 0, 1, None) == 0
    assert lib.wq8_prepared_values(None, None, None, None, 4, 64, 0, 3, None) == -1 and lib.wq8_prepared_values(None, None, None, None, 4, 60, 0, 1, None) == -2
    route = lambda tokens=4, experts=8, k=64, top=2, dtype=1, score=0: lib.wq8_route(None, k, dtype, None, 1, None, tokens, experts, k, top, score, 1, 1.0, None, None,
                                                                                      None, None)
    assert route(tokens=0) == 0
    assert [route(dtype=3), route(score=2)] == [-1] * 2
    assert [route(experts=0), route(experts=1025), route(k=60), route(top=0), route(top=9), route(tokens=65535 * 16 + 1), route(tokens=-1)] == [-2] * 7
    experts = lambda tokens=4, top=2, count=8, k=64, hidden=32, dtype=1, ldx=64: lib.wq8_experts(None, ldx, dtype, None, None, None, None, None, None, None, 0, None, None, k,
                                                                                                tokens, top, count, k, hidden, None, None)
    assert experts(tokens=0) == 0
    assert experts(dtype=2) == -1
    assert [experts(tokens=2049), experts(top=0), experts(count=0), experts(k=72), experts(hidden=24), experts(k=32768, hidden=32768), experts(ldx=2 ** 30),
            experts(tokens=-1)] == [-2] * 8
    sample = lambda rows=2, vocabulary=100, dtype=2: lib.wq8_sample(None, vocabulary, dtype, None, None, 1.0, None, 0, None, 1.0, None, 0.0, rows, vocabulary, None, None, None)
    assert sample(rows=0) == 0
    assert sample(dtype=3) == -1 and [sample(rows=-1), sample(rows=2 ** 17 + 1), sample(vocabulary=0), sample(vocabulary=2 ** 24 + 1)] == [-2] * 4


@pytest.mark.parametrize("given,kept", [(2 ** 32 + 3, 9), (2 ** 31, 9), (-2 ** 32 + 1, 9), (-2 ** 31 - 1, 9), (-2 ** 40 + 8, 9), (-1, 9), (0, 9), (9, 9), (7, 7)])
def test_numbers_of_top_k_beyond_32_bits(monkeypatch, given, kept):
    """How many of 9 tokens the C interface keeps, whose top_k has 32 bits, by what sample() hands to it."""
    import ctypes
    from types import SimpleNamespace

    from wgpkernels_amd.int8 import _native, _sample
    calls = []
    monkeypatch.setattr(_sample, "_check_devices", lambda *tensors: None)
    monkeypatch.setattr(_sample, "_layouts", _sample.Layouts())
    monkeypatch.setattr(_native, "gpu", lambda x: SimpleNamespace(index=0, stream=lambda: None))
    monkeypatch.setattr(_native, "call_on", lambda library, index, name, *args: calls.append((name, args)))
    wq.sample(torch.zeros(3, 9), torch.zeros(3), top_k=given)
    (name, args), = calls
    # logits, pitch, type, draws, then an address and a number of each option: temperature, top_k
    assert name == "wq8_sample" and args[6] is None
    top_k = ctypes.c_int(args[7]).value
    assert (top_k if 0 < top_k < 9 else 9) == kept


def test_workspace_of_a_sample():
    """A row's state, and a list of keys that is no longer than the vocabulary; never more than the query for any vocabulary says."""
    import ctypes
    lib, sizes, most = wq.library(), (ctypes.c_int64 * 2)(), (ctypes.c_int64 * 2)()
    lib.wq8_sample_workspace_for(1, 1, sizes)
    state = sizes[1]
    assert 14000 < state < 16384 and state % 16 == 0
    for rows, vocabulary, keys in ((1, 131072, 16384), (1024, 300, 300), (8192, 20000, 16384), (16384, 20000, 8192), (16384, 5000, 5000), (2 ** 17, 300, 300), (2 ** 17, 2 ** 24, 2048)):
        lib.wq8_sample_workspace_for(rows, vocabulary, sizes)
        lib.wq8_sample_workspace(rows, most)
        assert list(sizes) == [rows * (state + 8 * keys), rows * state] and sizes[0] <= most[0]
    for rows, vocabulary in ((0, 100), (-1, 100), (5, 0)):
        lib.wq8_sample_workspace_for(rows, vocabulary, sizes)
        assert list(sizes) == [0, 0]
