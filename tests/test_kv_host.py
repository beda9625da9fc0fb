"""The rotary and 8-bit cache operators without a GPU: what they refuse, before anything is launched, and how a rotary plan holds
its angles."""
import math

import pytest
import torch

from wgpkernels_amd import int8 as wq


def cache(pages=4, heads=2, block=16, head_dim=64, device="cpu"):
    return wq.KVCache(pages, heads, head_dim, block, device=device)


def rows(tokens=3, heads=2, head_dim=64, dtype=torch.bfloat16):
    return torch.zeros(tokens, heads, head_dim, dtype=dtype)


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype)


# ---- rotary --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sections", [(), (0,), (4, -1), (1, 1, 1, 1)])
def test_plan_refuses_sections(sections):
    with pytest.raises(ValueError):
        wq.rotary_plan(sections, device="cpu")


@pytest.mark.parametrize("options", [{"style": "thirds"}, {"ladder": "steps"}, {"base": 0.0}, {"base": math.inf}, {"frequencies": [1.0]},
                                     {"frequencies": [1.0, math.nan, 0.5, 0.1]}])
def test_plan_refuses_options(options):
    with pytest.raises(ValueError):
        wq.rotary_plan((4,), device="cpu", **options)


@pytest.mark.parametrize("ladder", ["axis", "joint"])
def test_plan_turns(ladder):
    """position * turns modulo 2^64 is the angle, at positions where 32-bit angles are lost. A frequency in FP64 is off by at most
    2^-53 of itself, the turns by 2^-53 (two operations) and 2^-65: at |position| < 2^31 the angle by less than 2^-20 turns."""
    sections = (5, 4, 7)
    plan = wq.rotary_plan(sections, ladder=ladder, base=500000.0, device="cpu")
    assert plan.pairs == 16 and plan.axis.tolist() == [0] * 5 + [1] * 4 + [2] * 7
    at = 0
    for n in sections:
        for i in range(n):
            exponent = i / n if ladder == "axis" else at / 16
            for position in (0, 1, -1, 4097, 1_000_003, -(2 ** 31) + 1):
                angle = math.fmod(position * 500000.0 ** -exponent / (2 * math.pi), 1.0)
                held = (position * plan.turns[at].item()) % 2 ** 64 / 2 ** 64
                off = (held - angle) % 1.0
                assert min(off, 1 - off) < 2.0 ** -20, (at, position)
            at += 1


def test_plan_takes_any_frequency():
    plan = wq.rotary_plan((3,), frequencies=[-0.25, 2 * math.pi * 3, 7.5], device="cpu")
    turns = [t / 2 ** 64 for t in plan.turns.tolist()]
    for t, f in zip(turns, (-0.25, 2 * math.pi * 3, 7.5)):
        off = (t - f / (2 * math.pi)) % 1.0
        assert min(off, 1 - off) < 1e-14


@pytest.mark.parametrize("change", ["type", "mixed", "tokens", "width", "strides", "aligned", "wide", "positions", "position_type", "many", "outs", "cpu"])
def test_rotary_refuses(change):
    plan = wq.rotary_plan((16, 16), device="cpu")
    q, k, positions, out = rows(), rows(heads=1), torch.zeros(3, 2, dtype=torch.int32), None
    if change == "type":
        q, k = q.double(), k.double()
    elif change == "mixed":
        k = k.half()
    elif change == "tokens":
        k = rows(4, 1)
    elif change == "width":
        q, k = rows(head_dim=68), rows(head_dim=68)
    elif change == "strides":
        q = torch.zeros(3, 64, 2, dtype=torch.bfloat16).transpose(1, 2)
    elif change == "aligned":
        q = torch.zeros(3, 2, 68, dtype=torch.bfloat16)[..., :64]
    elif change == "wide":
        plan = wq.rotary_plan((33,), device="cpu")
        positions = torch.zeros(3, dtype=torch.int32)
    elif change == "positions":
        positions = torch.zeros(3, 3, dtype=torch.int32)
    elif change == "position_type":
        positions = positions.float()
    elif change == "many":
        with pytest.raises(ValueError):
            wq.rotary((q, q, q, q, q), positions, plan)
        q = ()
        with pytest.raises(ValueError):
            wq.rotary(q, positions, plan)
        return
    elif change == "outs":
        out = (torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros_like(k))
    with pytest.raises(ValueError):
        wq.rotary((q, k), positions, plan, out=out)


# ---- the cache -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(4, 2, 24, 64), (4, 2, 16, 60), (4, 2, 16, 2048)])
def test_cache_refuses_shapes(shape):
    with pytest.raises(ValueError):
        wq.KVCache(shape[0], shape[1], shape[3], shape[2], device="cpu")


def test_cache_refuses_no_heads():
    with pytest.raises(ValueError, match="head"):
        cache(heads=0)


def test_cache_refuses_parts():
    good = cache()
    k, ks, v, vs = good.k_codes, good.k_scales, good.v_codes, good.v_scales
    assert wq.KVCache.from_codes(k, ks, v, vs).k_codes is k
    bad = [(k.float(), ks, v, vs), (k, ks.double(), v, vs), (k, ks[:2], v, vs), (k, ks, v[:2], vs), (k, ks.t().contiguous().t(), v, vs),
           (k.transpose(1, 2).contiguous().transpose(1, 2), ks, v, vs), (k[0], ks, v[0], vs)]
    for parts in bad:
        with pytest.raises(ValueError):
            wq.KVCache.from_codes(*parts)


def test_plan_refuses():
    past, new, tables, free, used = ints(3, 4), ints(1, 1), torch.zeros(2, 5, dtype=torch.int32), ints(1, 2, 3), ints(0)
    bad = [(past.long(), new, tables, free, used, 16, 2), (past, ints(1), tables, free, used, 16, 2), (past, new, tables.long(), free, used, 16, 2),
           (past, new, tables.t(), free, used, 16, 2), (past, new, tables[:1], free, used, 16, 2), (past, new, tables, free.float(), used, 16, 2),
           (past, new, tables, free, ints(0, 0), 16, 2), (past, new, tables, free, used, 0, 2), (past, new, tables, free, used, 16, -1),
           (past, new, tables, free, used, 16, 2)]  # the last: nothing wrong but the device
    for args in bad:
        with pytest.raises(ValueError):
            wq.kv_plan(*args)


def test_write_and_read_refuse():
    c, slots = cache(), ints(0, 1, 2, dtype=torch.int64)
    k = rows()
    for args in [(k, rows(heads=3), slots), (rows(heads=3), rows(heads=3), slots), (k, k.half(), slots), (k, k, slots.int()), (k, k, slots[:2]),
                 (k.double(), k.double(), slots), (k[..., :32], k[..., :32], slots), (k, k, slots)]:
        with pytest.raises(ValueError):
            wq.kv_write(c, *args)
    for args in [(slots.int(),), (slots, torch.float64), (slots,)]:
        with pytest.raises(ValueError):
            wq.kv_read(c, *args)


def test_attention_refuses():
    c, tables, lens, starts, q = cache(), torch.zeros(2, 3, dtype=torch.int32), ints(3, 4), ints(0, 1, 3), rows(heads=4)
    bad = [((q.float(), c, tables, lens, starts), {}), ((rows(heads=3), c, tables, lens, starts), {}), ((rows(heads=4, head_dim=128), c, tables, lens, starts), {}),
           ((rows(heads=4, head_dim=72), cache(head_dim=72), tables, lens, starts), {}), ((q, c, tables[:1], lens, starts), {}),
           ((q, c, tables.long(), lens, starts), {}), ((q, c, tables, lens.long(), starts), {}), ((q, c, tables, lens, starts[:2]), {}),
           ((q, c, tables, lens, starts), {"window": -1}), ((q, c, tables, lens, starts), {"out": q[:2]}), ((q, c, tables, lens, starts), {"out": q.half()}),
           ((q, c, tables, lens, starts), {})]
    for args, options in bad:
        with pytest.raises(ValueError):
            wq.kv_attention(*args, **options)


def test_c_entries_refuse():
    """Negative codes before any launch, for callers of the C-ABI."""
    import ctypes
    lib = wq._native.Library(wq.default_library_path())
    two, four = (ctypes.c_void_p * 2)(), (ctypes.c_longlong * 10)(*[1] * 10)
    rotary = lambda **o: lib.wq8_rotary(two, two, four, o.get("count", 2), None, 1, 1, 0, o.get("tokens", 4), None, None, o.get("pairs", 8),
                                        o.get("head_dim", 64), o.get("style", 0), 0, o.get("dtype", 1), None)
    assert rotary(dtype=3) == rotary(style=2) == -1
    assert rotary(count=5) == rotary(tokens=-1) == rotary(pairs=33) == rotary(head_dim=60) == -2
    assert rotary(tokens=0) == 0
    plan = lambda **o: lib.wq8_kv_plan(None, None, None, 1, None, o.get("free", 0), None, o.get("requests", 1), o.get("width", 1), o.get("block", 16),
                                       o.get("tokens", 1), None, None, None, None, None, None, None)
    assert plan(free=-1) == plan(requests=-1) == plan(width=-1) == plan(block=0) == plan(tokens=-1) == plan(tokens=2 ** 31) == -2
    write = lambda **o: lib.wq8_kv_write(None, None, four, None, o.get("tokens", 1), None, None, None, None, o.get("pages", 4), o.get("heads", 2), o.get("block", 16),
                                         o.get("head_dim", 64), o.get("dtype", 1), None, None)
    assert write(dtype=3) == -1
    assert write(block=256) == write(head_dim=12) == write(heads=0) == write(tokens=-1) == write(pages=-1) == -2
    assert write(tokens=0) == 0
    read = lambda **o: lib.wq8_kv_read(None, None, None, None, None, o.get("tokens", 1), None, None, 4, 2, o.get("block", 16), 64, o.get("dtype", 1), None)
    assert read(dtype=-1) == -1 and read(block=0) == -2 and read(tokens=0) == 0
    attend = lambda **o: lib.wq8_kv_attention(None, None, four, None, None, None, None, None, 1, 1, None, None, o.get("tokens", 1), o.get("requests", 1),
                                              o.get("heads", 2), o.get("group", 1), o.get("head_dim", 64), o.get("block", 16), 4, 1.0, 1, o.get("window", 0),
                                              o.get("dtype", 1), 256, None, None)
    assert attend(dtype=2) == -1
    assert attend(head_dim=80) == attend(block=24) == attend(heads=0) == attend(group=0) == attend(window=-1) == attend(tokens=-1) == -2
    assert attend(tokens=0) == attend(requests=0) == 0


@pytest.mark.parametrize("options", [{"base": 500000.0}, {"base": 500000.0, "ladder": "joint"}, {"base": 1e-300},
                                     {"frequencies": [1.0, -0.3, 2 * math.pi * 3, 1e300, 5e-324, 0.0, 1e-9, 123456.789, 2.0 ** 1000]}])
def test_plan_turns_at_far_positions(options):
    """A pair's turns are the nearest fraction of 2^64 to its FP64 frequency over 2 pi, so that the angle of position p is off by
    |p| 2^-65 turns and no more; against 2 pi from another series, in as many digits as 2^1024 and 2^62 leave."""
    from decimal import Decimal, localcontext
    from fractions import Fraction
    plan = wq.rotary_plan((4, 5), device="cpu", **options)
    steps = [i / 9 for i in range(9)] if options.get("ladder") == "joint" else [i / 4 for i in range(4)] + [i / 5 for i in range(5)]
    frequencies = options.get("frequencies") or [options["base"] ** -s for s in steps]
    with localcontext() as c:
        c.prec = 420
        held, t, n, na, d, da, pi = 0, Decimal(3), 1, 0, 0, 24, Decimal(3)  # pi = 6 arcsin(1 / 2)
        while held != pi:
            held, n, na, d, da = pi, n + na, na + 8, d + da, da + 32
            t = t * n / d
            pi += t
        two_pi = 2 * Fraction(pi)
    for f, turns in zip(frequencies, plan.turns.tolist()):
        for position in (1, -1, 4097, 2 ** 31 - 1, -(2 ** 40) + 3, 2 ** 50 + 1, -(2 ** 62) + 5):
            off = (Fraction(position * turns, 2 ** 64) - position * Fraction(f) / two_pi) % 1
            assert min(off, 1 - off) <= abs(position) * Fraction(1, 2 ** 65), (f, position)


def test_written_rows_do_not_overlap():
    """Rows that several workgroups would write at once: block tables completed in place, outputs given by the caller."""
    from wgpkernels_amd.int8._rotary import _check_written
    past, new, free, used = ints(3, 4), ints(1, 1), ints(1, 2, 3), ints(0)
    one = torch.zeros(5, dtype=torch.int32)
    for tables in (one.expand(2, 5), torch.zeros(8, dtype=torch.int32).as_strided((2, 5), (3, 1))):
        with pytest.raises(ValueError, match="overlap"):
            wq.kv_plan(past, new, tables, free, used, 16, 2)
    good = torch.zeros(6, 4, 8)
    for rows_ in (good, good[:, 1:3], good.transpose(0, 1), good[::2, ::3], good[:1].expand(1, 4, 8), good[:0], torch.zeros(6, 1, 8), torch.zeros(1, 8).expand(0, 4, 8)):
        _check_written(rows_, "outputs")
    for rows_ in (good[:1].expand(6, 4, 8), good[:, :1].expand(6, 4, 8), good.as_strided((6, 4, 8), (24, 8, 1)), good.as_strided((6, 4, 8), (32, 4, 1))):
        with pytest.raises(ValueError, match="overlap"):
            _check_written(rows_, "outputs")
