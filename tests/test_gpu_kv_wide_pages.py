"""Writes of pages of 16384 values and more: kept in registers up to 32768 values, read again above."""
import math

import pytest
import torch

import test_gpu_kv
from test_gpu_kv import held, ints, step_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("head_dim,block", [(128, 128), (256, 128), (1024, 32), (512, 128), (1024, 128), (328, 128)])
@pytest.mark.parametrize("tokens", [1, 200, 700])
@pytest.mark.parametrize("order", ["run", "any"])
def test_write(wq, dtype, tokens, head_dim, block, order):
    test_gpu_kv.test_write(wq, dtype, tokens, 2, head_dim, block, order)


@pytest.mark.parametrize("tokens", [3, 600])
@pytest.mark.parametrize("head_dim", [256, 1024])
def test_values_that_are_not_finite(wq, head_dim, tokens):
    """NaN is held as zero and an infinity as the largest finite number beside which the page's others come to 0; the other head keeps its values."""
    block = 128
    pages = -(-tokens // block) + 1
    cache = wq.KVCache(pages, 2, head_dim, block)
    g = torch.Generator(device="cuda").manual_seed(head_dim)
    k = torch.randn(tokens, 2, head_dim, generator=g, device="cuda").bfloat16()
    slots = torch.arange(tokens, device="cuda") + block
    bad = k.clone()
    bad[0, 0, 5], bad[2, 1, 3] = math.nan, -math.inf
    wq.kv_write(cache, bad, k, slots)
    assert torch.isfinite(cache.k_scales).all()
    page, at = slots // block, slots % block
    got = held(cache, "k")[page, :, at]
    want = k.double()
    want[0, 0, 5] = 0.0
    ok = torch.ones(tokens, 2, dtype=torch.bool, device="cuda")
    ok[:block, 1] = False  # beside the infinity
    scales = cache.k_scales[page]
    assert ((got - want).abs().amax(2) <= step_of(scales))[ok].all()
    assert got[0, 0, 5] == 0 and abs(got[2, 1, 3].item() / -torch.finfo(torch.float32).max - 1) < 2 ** -20
    rest = got[:block, 1].clone()
    rest[2, 3] = 0.0
    assert not rest.any()
    assert ((held(cache, "v")[page, :, at] - k.double()).abs().amax(2) <= step_of(cache.v_scales[page])).all()


def test_growing_page_read_again(wq):
    """A page of 131072 values that goes on, its scale growing with every token: what it holds is coded again each time."""
    cache = wq.KVCache(2, 1, 1024, 128)
    cache.k_scales.fill_(5.0)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(16, 1, 1024, generator=g, device="cuda") * torch.arange(1, 17, device="cuda")[:, None, None]
    for t in range(16):
        wq.kv_write(cache, x[t:t + 1], x[t:t + 1], ints([128 + t], torch.int64))
    scale = (x.abs().max().double() / 127).float()
    assert cache.k_scales[1].item() == scale.item() and cache.k_scales[0].item() == 5.0
    off = (held(cache, "k")[1, 0, :16] - x[:, 0].double()).abs().amax(1)
    grown = torch.tensor([len({x[:j + 1].abs().max().item() for j in range(t, 16)}) for t in range(16)], device="cuda")
    assert (off <= step_of(scale) * grown).all()
