"""Attention over the 8-bit cache where a workgroup's part passes 4096 keys (pages and scales come 64 at a time and are loaded again), where
prompts and single tokens share a call, and over windows without causality; against 64 bits.

Tolerance, as in test_gpu_kv_attention.py: half a step of the output; 2^-11 of sum p |v| for weights in FP16; 2^-25 of every key at the largest
value for those below FP16's normal range; and for the scores, FP32 sums of head_dim products in any order, 2 head_dim 2^-24
of the largest sum |q k| scale (a weight and the weights' sum each move by the score's error)."""
import ctypes
import math
import random

import pytest
import torch

from test_gpu_kv_attention import ints, make, rows, starts_of

pytestmark = pytest.mark.gpu


def exact(q, cache, tables, lens, new, causal, window):
    """Rows and the bound of their error but for the output's rounding."""
    q, heads, block, d = q.cpu().double(), cache.heads, cache.block, cache.head_dim
    group = q.shape[1] // heads
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        if m and n:
            position = torch.arange(n)
            page, off = tables[r].cpu()[position // block].long(), position % block
            k, v = (c.cpu()[page, :, off].double() * s.cpu()[page].double()[..., None]
                    for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
            k, v = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()  # (heads, d, keys), (heads, keys, d)
            x = q[at:at + m].reshape(m, heads, group, d).permute(1, 0, 2, 3).reshape(heads, m * group, d)
            own = n - m + torch.arange(m * group)[:, None] // group
            hidden = torch.zeros(m * group, n, dtype=torch.bool)
            if causal:
                hidden |= position > own
            if window:
                hidden |= position <= own - window
            s = torch.matmul(x, k).mul_(d ** -0.5).masked_fill_(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))  # a row that sees nothing
            scores = 2 * d * 2.0 ** -24 * torch.matmul(x.abs(), k.abs()).mul_(d ** -0.5).masked_fill_(hidden, 0.0).amax(-1, keepdim=True)
            seen = (~hidden).sum(-1, keepdim=True)
            off = (2.0 ** -11 + scores) * torch.matmul(p, v.abs()) + 2.0 ** -25 * seen * v.abs().amax((1, 2), keepdim=True)
            back = lambda t: t.reshape(heads, m, group, d).permute(1, 0, 2, 3).reshape(m, heads * group, d)
            out[at:at + m], bound[at:at + m] = back(torch.matmul(p, v)), back(off)
        at += m
    return out, bound


def check(got, q, cache, tables, lens, new, causal=True, window=0):
    want, bound = exact(q, cache, tables, lens, new, causal, window)
    info = torch.finfo(got.dtype)
    bound += info.eps / 2 * want.abs().clamp(min=info.smallest_normal)
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max().item()


def attention_on(wq, workgroups, q, cache, tables, lens, starts, causal=True, window=0):
    """kv_attention with the work split as for a GPU of so few compute units: long parts from small inputs."""
    lib, out = wq.library(), torch.empty_like(q)
    heads, group = cache.heads, q.shape[1] // cache.heads
    sizes = (ctypes.c_int64 * 2)()
    lib.wq8_kv_attention_workspace(q.shape[0], lens.shape[0], heads, group, cache.head_dim, workgroups, sizes)
    workspace = torch.empty(sizes[0], dtype=torch.int8, device="cuda")
    strides = (ctypes.c_longlong * 4)(q.stride(0), q.stride(1), out.stride(0), out.stride(1))
    lib.call("wq8_kv_attention", q.data_ptr(), out.data_ptr(), strides, cache.k_codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(),
             cache.v_scales.data_ptr(), tables.data_ptr(), tables.stride(0), tables.shape[1], lens.data_ptr(), starts.data_ptr(), q.shape[0], lens.shape[0], heads,
             group, cache.head_dim, cache.block, cache.pages, cache.head_dim ** -0.5, causal, window, wq.DTYPES[q.dtype], workgroups, workspace.data_ptr(),
             torch.cuda.current_stream().cuda_stream)
    return out


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("new,group", [(1, 6), (40, 1)], ids=["few", "many"])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 9500)])
def test_parts_of_many_keys(wq, head_dim, block, new, group, causal, window):
    """Half the rows look for one key each (at and around multiples of 4096 of its part and anywhere), so that a wrong page shows as another value."""
    print(f"parts of many keys {head_dim} {block} {new} {group} {causal} {window}", flush=True)
    heads, length = 8, 20011
    cache, tables = make(wq, [length], heads, head_dim, block, head_dim)
    g = torch.Generator(device="cuda").manual_seed(block)
    cache.k_scales.uniform_(0.010, 0.012, generator=g)
    q = rows(new, heads * group, head_dim, torch.bfloat16, 31).float()
    rng = random.Random(head_dim + block)
    wanted = [0, 4095, 4096, 4097, 8191, 8192, 8193, 12288, 16383, 16384, length - 1 - new, 10005, 14100, 14101]
    # a sum of |q k| scale of 64 and less; other keys' scores are 20 and more below it
    size = {64: 12.0, 128: 6.0, 256: 4.0}[head_dim]
    for i in range(0, new * heads * group, 2):
        token, head = i // (heads * group), i % (heads * group)
        key = wanted[i // 2] if i // 2 < len(wanted) else rng.randrange(length - new)
        code = cache.k_codes[tables[0, key // block].long(), head // group, key % block]
        q[token, head] = size * torch.sign(code.float())
    q = q.bfloat16()
    for got in (attention_on(wq, 8, q, cache, tables, ints([length]), starts_of([new]), causal, window),
                wq.kv_attention(q, cache, tables, ints([length]), starts_of([new]), causal=causal, window=window)):
        check(got, q, cache, tables, [length], [new], causal, window)


@pytest.mark.parametrize("head_dim,block", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("lens,new,group", [([700] + [40 + 31 * i for i in range(50)], [600] + [1] * 50, 1),  # 13 rows a request on average
                                            ([900, 3, 1300, 64, 500], [900, 1, 2, 0, 1], 4),  # 723
                                            ([500, 2000, 1, 333, 800, 0], [300, 1, 1, 1, 2, 0], 1),  # 51
                                            ([1, 640], [1, 600], 5)], ids=["few", "many", "both", "last"])
def test_prompts_beside_single_tokens(wq, head_dim, block, lens, new, group):
    print(f"prompts beside single tokens {head_dim} {block} {len(lens)} {group}", flush=True)
    cache, tables = make(wq, lens, 2, head_dim, block, len(lens))
    q = rows(sum(new), 2 * group, head_dim, torch.float16, 41)
    for causal, window in ((True, 0), (False, 0), (True, 100)):
        got = wq.kv_attention(q, cache, tables, ints(lens), starts_of(new), causal=causal, window=window)
        check(got, q, cache, tables, lens, new, causal, window)


@pytest.mark.parametrize("lens,new,window", [([2300], [2300], 100), ([1500, 700, 40], [1500, 200, 40], 333), ([2000], [1], 64)])
def test_window_without_causality(wq, lens, new, window):
    """Rows see from the window's start to their request's end: the first tiles many keys, the last ones few."""
    cache, tables = make(wq, lens, 3, 64, 32, 51)
    q = rows(sum(new), 3, 64, torch.bfloat16, 52)
    for workgroups in (8, 64, 256):
        got = attention_on(wq, workgroups, q, cache, tables, ints(lens), starts_of(new), False, window)
        check(got, q, cache, tables, lens, new, False, window)


def test_overlapping_outputs_are_refused(wq):
    """Before any launch: rows that several workgroups would write at once."""
    lens, new = [70, 20], [3, 2]
    cache, tables = make(wq, lens, 2, 64, 32, 61)
    q = rows(5, 4, 64, torch.bfloat16, 62)
    for out in (q[:1].clone().expand(5, 4, 64), q[:, :1].clone().expand(5, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            wq.kv_attention(q, cache, tables, ints(lens), starts_of(new), out=out)
        with pytest.raises(ValueError, match="overlap"):
            wq.rotary(q, torch.arange(5, device="cuda"), wq.rotary_plan((4,)), out=out)
    out = torch.empty(4, 5, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)  # heads first
    assert wq.kv_attention(q, cache, tables, ints(lens), starts_of(new), out=out) is out
    assert torch.equal(out, wq.kv_attention(q, cache, tables, ints(lens), starts_of(new)))
