"""The paged 8-bit key/value cache on MI355X: planned on the GPU from request lengths, written, read and attended over.

Keys and values are held as INT8 codes (pages, heads, block, head_dim) with one FP32 scale per page and head: a value is
code * scale, scale = the largest magnitude of the page's tokens / 127. A slot is page * block + the place in the page. A
request's tokens lie on the pages that its row of a block table names, in order.

    plan = kv_plan(past, new, tables, free, used, block, tokens)      # slots, positions, block tables of a step
    kv_write(cache, k, v, plan.slots)                                  # append the step's keys and values
    out = kv_attention(q, cache, tables, plan.lens, plan.starts)       # the step's queries over the cache

None of these waits for the GPU or reads lengths on the host: a step can be captured in a HIP graph.
"""
import ctypes
from typing import NamedTuple

import torch

from . import DTYPES, _native, library
from ._rotary import Layouts, _check_aligned, _check_devices, _check_rows, _check_written

BLOCKS = (16, 32, 64, 128)
ATTENTION_HEAD_DIMS = (64, 128, 256)


class KVPlan(NamedTuple):
    """What kv_plan() gives for a step of `tokens` tokens and R requests."""
    slots: torch.Tensor      # (tokens,) int64: where each token goes, -1 for those that go nowhere
    positions: torch.Tensor  # (tokens,) int32: its position in its request
    starts: torch.Tensor     # (R + 1,) int32: each request's first token in the step
    lens: torch.Tensor       # (R,) int32: each request's length after the step
    used: torch.Tensor       # (1,) int32: pages of the free list taken so far
    missing: torch.Tensor    # (1,) int32: requests that found no room


class KVCache:
    """An empty cache of `pages` pages of `block` tokens (16, 32, 64 or 128) on a GPU."""
    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "owner", "layouts")

    def __init__(self, pages, heads, head_dim, block=64, device="cuda"):
        codes = lambda: torch.zeros(pages, heads, block, head_dim, dtype=torch.int8, device=device)
        scales = lambda: torch.zeros(pages, heads, dtype=torch.float32, device=device)
        self._take(codes(), scales(), codes(), scales())

    @classmethod
    def from_codes(cls, k_codes, k_scales, v_codes, v_scales):
        """A cache over existing codes (pages, heads, block, head_dim) int8 and scales (pages, heads) float32, not copied. Scales
        are finite and not negative; where one is zero, so are its codes."""
        cache = cls.__new__(cls)
        cache._take(k_codes, k_scales, v_codes, v_scales)
        return cache

    def _take(self, k_codes, k_scales, v_codes, v_scales):
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape or k_codes.shape[2] not in BLOCKS or k_codes.shape[3] % 8 or not 8 <= k_codes.shape[3] <= 1024:
            raise ValueError(f"cache codes must be (pages, heads, {' / '.join(map(str, BLOCKS))} tokens, a multiple of 8 channels), the same for keys and values")
        if not k_codes.shape[1]:
            raise ValueError("a cache needs heads")
        if k_codes.dtype != torch.int8 or v_codes.dtype != torch.int8 or k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32:
            raise ValueError("cache codes must be INT8, their scales FP32")
        if k_scales.shape != k_codes.shape[:2] or v_scales.shape != k_codes.shape[:2]:
            raise ValueError("cache scales must be (pages, heads)")
        parts = (k_codes, k_scales, v_codes, v_scales)
        if not all(t.is_contiguous() for t in parts) or k_codes.data_ptr() % 16 or v_codes.data_ptr() % 16:
            raise ValueError("cache codes and scales must be contiguous, the codes 16-byte aligned")
        if any(t.device != k_codes.device for t in parts):
            raise ValueError("cache codes and scales must be on one device")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = parts
        self.layouts = Layouts()
        # which token of a kv_write() call each slot takes: scratch of that call (entries are checked, never cleared)
        self.owner = torch.empty(k_codes.shape[0] * k_codes.shape[2], dtype=torch.int32, device=k_codes.device)

    pages = property(lambda self: self.k_codes.shape[0])
    heads = property(lambda self: self.k_codes.shape[1])
    block = property(lambda self: self.k_codes.shape[2])
    head_dim = property(lambda self: self.k_codes.shape[3])


def _check_ints(t, name, dtype=torch.int32, dim=1):
    if t.dtype != dtype or t.dim() != dim or (t.numel() and not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dim}-D {str(dtype).removeprefix('torch.')} tensor")


def _check_tables(tables):
    if tables.dtype != torch.int32 or tables.dim() != 2 or (tables.shape[1] > 1 and tables.stride(1) != 1):
        raise ValueError("block tables must be (requests, pages) int32 with unit column stride")


def kv_plan(past, new, tables, free, used, block, tokens):
    """Slots, positions and block tables of a step in which request r, with past[r] tokens cached, brings new[r] more: new tokens
    stand one request after another in rows of the step's `tokens` (padding beyond their sum gets slot -1, position 0).

    past, new: (R,) int32 (negative counts as 0). tables: (R, width) int32, completed in place with the pages that the new tokens
    begin: free[used], free[used + 1], ... in the order of requests and tokens. free: (F,) int32; used: (1,) int32. A request that
    the table's width, `tokens`, 31-bit positions or the free pages left cannot hold gets no page, slots -1 and its old length, and so does
    every later one that needs a page where the free list ran out. Everything is int32 / int64 on the GPU; nothing is read
    on the host."""
    key = (past.shape, past.dtype, past.stride(), new.shape, new.dtype, new.stride(), free.shape, free.dtype, free.stride(), tables.shape, tables.stride(),
           tables.dtype, used.shape, used.dtype, block, tokens, past.get_device(), new.get_device(), free.get_device(), tables.get_device(), used.get_device())
    splits = _plan_layouts.get(key) or _plan_layouts.keep(key, _check_plan(past, new, tables, free, used, block, tokens))
    slots = past.new_empty(tokens, dtype=torch.int64)
    held = past.new_empty(tokens + 2 * splits[2] + 3)
    positions, starts, lens, used_out, missing = held.split_with_sizes(splits)
    requests, at = splits[2], held.data_ptr()
    starts_at = at + 4 * tokens
    lens_at = starts_at + 4 * requests + 4
    used_at = lens_at + 4 * requests
    library().call("wq8_kv_plan", past.data_ptr(), new.data_ptr(), tables.data_ptr(), tables.stride(0), free.data_ptr(), free.shape[0], used.data_ptr(),
                   requests, tables.shape[1], block, tokens, slots.data_ptr(), at, starts_at, lens_at, used_at, used_at + 4, _native.gpu(past).stream())
    return KVPlan(slots, positions, starts, lens, used_out, missing)


_plan_layouts = Layouts()


def _check_plan(past, new, tables, free, used, block, tokens):
    """Lengths of a plan's int32 results."""
    _check_ints(past, "past")
    _check_ints(new, "new")
    _check_ints(free, "free")
    _check_tables(tables)
    if used.dtype != torch.int32 or used.numel() != 1:
        raise ValueError("used must be one int32")
    requests = past.shape[0]
    if new.shape[0] != requests or tables.shape[0] != requests:
        raise ValueError(f"past, new and tables must be of as many requests, not {requests}, {new.shape[0]} and {tables.shape[0]}")
    if requests > 1 and tables.stride(0) < tables.shape[1]:
        raise ValueError("rows of block tables must not overlap: they are completed in place")
    if not 1 <= block <= 2 ** 30 or not 0 <= tokens < 2 ** 31:
        raise ValueError("a block of 1 to 2^30 tokens and a token count are wanted")
    _check_devices(past, new, tables, free, used)
    return [tokens, requests + 1, requests, 1, 1]


def _check_write(cache, k, v, slots):
    _check_rows(k, "keys")
    _check_rows(v, "values")
    _check_ints(slots, "slots", torch.int64)
    if k.shape != v.shape or k.dtype != v.dtype or k.shape[1:] != (cache.heads, cache.head_dim) or slots.shape[0] != k.shape[0]:
        raise ValueError(f"keys and values must be (tokens, {cache.heads}, {cache.head_dim}), of one type, with a slot each")
    _check_devices(cache.k_codes, k, v, slots)
    return (ctypes.c_longlong * 4)(k.stride(0), k.stride(1), v.stride(0), v.stride(1)), k.shape[0], DTYPES[k.dtype], (cache.pages, cache.heads, cache.block, cache.head_dim)


def kv_write(cache, k, v, slots):
    """Keys and values (tokens, heads, head_dim), BF16, FP16 or FP32, into the cache at `slots` (int64; any order, each at most once;
    those outside the cache, as -1, are left out). A page's scale grows to its largest value, and tokens that it holds are then
    coded again; a write to its first slot begins it anew. NaN is held as 0 and infinities as the largest finite number (beside
    which the other tokens of the page come to 0)."""
    key = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), slots.shape, slots.stride(), slots.dtype,
           slots.get_device())
    strides, tokens, dtype, shape = cache.layouts.get(key) or cache.layouts.keep(key, _check_write(cache, k, v, slots))
    codes = cache.k_codes
    k_at, v_at = k.data_ptr(), v.data_ptr()
    _check_aligned((k_at, v_at))
    library().call("wq8_kv_write", k_at, v_at, strides, slots.data_ptr(), tokens, codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(),
                   cache.v_scales.data_ptr(), *shape, dtype, cache.owner.data_ptr(), _native.gpu(codes).stream())


def kv_read(cache, slots, dtype=torch.bfloat16):
    """The keys and values at `slots` (int64; zeros outside the cache), rounded once to dtype: two (tokens, heads, head_dim) tensors."""
    key = (slots.shape, slots.stride(), slots.dtype, slots.get_device(), dtype)
    shape, like = cache.layouts.get(key) or cache.layouts.keep(key, _check_read(cache, slots, dtype))
    codes = cache.k_codes
    k = codes.new_empty(like, dtype=dtype)
    v = torch.empty_like(k)
    library().call("wq8_kv_read", codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(), cache.v_scales.data_ptr(), slots.data_ptr(), like[0],
                   k.data_ptr(), v.data_ptr(), *shape, DTYPES[dtype], _native.gpu(codes).stream())
    return k, v


def _check_read(cache, slots, dtype):
    _check_ints(slots, "slots", torch.int64)
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be FP16, BF16 or FP32, not {dtype}")
    _check_devices(cache.k_codes, slots)
    return (cache.pages, cache.heads, cache.block, cache.head_dim), (slots.shape[0], cache.heads, cache.head_dim)




def kv_attention(q, cache, tables, lens, starts, causal=True, window=0, scale=None, out=None):
    """Attention of the step's queries over the cache: q (tokens, query heads, head_dim) BF16 or FP16, head_dim 64, 128 or 256, each key/value
    head serving query heads / heads of them, in order. Request r owns rows starts[r] to starts[r + 1] (int32, not
    decreasing) and sees the first lens[r] (int32) tokens of its row of `tables`, its own rows being the last of them. out: a tensor of
    q's shape and type whose rows do not overlap, nor share memory with q.

    causal: a row sees the tokens up to itself, otherwise all of its request's; window > 0: of those, the ones after
    position - window. scale: of the scores, 1 / sqrt(head_dim) by default. Rows that see nothing are zero; pages outside the cache are
    hidden; rows of no request are not written (uninitialised in a new output). Returns (tokens, query heads, head_dim) in q's dtype. Sums and
    the softmax's statistics are FP32, its weights FP16 relative to the largest; value scales below 2^-90 count as that (off by
    less than 2^-83). Not recorded for autograd."""
    key = (q.shape, q.stride(), q.dtype, q.get_device(), tables.shape, tables.stride(), tables.dtype, tables.get_device(), lens.shape, lens.stride(), lens.dtype,
           lens.get_device(), starts.shape, starts.stride(), starts.dtype, starts.get_device())
    layout = cache.layouts.get(key) or cache.layouts.keep(key, _check_attention(q, cache, tables, lens, starts))
    strides, table_stride, shape, default_scale, dtype, cus, workspace_bytes = layout
    if not 0 <= window < 2 ** 31:
        raise ValueError("the window must not be negative")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_rows(out, "outputs")
        _check_written(out, "outputs")
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("outputs do not match the queries")
        _check_devices(q, out)
        strides = type(strides)(strides[0], strides[1], out.stride(0), out.stride(1))
    codes = cache.k_codes
    q_at, out_at = q.data_ptr(), out.data_ptr()
    _check_aligned((q_at,))
    workspace = codes.new_empty(workspace_bytes) if workspace_bytes else None
    library().call("wq8_kv_attention", q_at, out_at, strides, codes.data_ptr(), cache.k_scales.data_ptr(), cache.v_codes.data_ptr(), cache.v_scales.data_ptr(),
                   tables.data_ptr(), table_stride, tables.shape[1], lens.data_ptr(), starts.data_ptr(), *shape, default_scale if scale is None else scale,
                   causal, window, dtype, cus, _native.ptr(workspace), _native.gpu(codes).stream())
    return out


def _check_attention(q, cache, tables, lens, starts):
    _check_rows(q, "queries")
    _check_ints(lens, "lens")
    _check_ints(starts, "starts")
    _check_tables(tables)
    tokens, q_heads, width = q.shape
    heads, head_dim, requests = cache.heads, cache.head_dim, lens.shape[0]
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"queries must be FP16 or BF16, not {q.dtype}")
    if width != head_dim or head_dim not in ATTENTION_HEAD_DIMS or not q_heads or q_heads % heads:
        raise ValueError(f"queries must have heads of {head_dim} channels ({', '.join(map(str, ATTENTION_HEAD_DIMS))}), a multiple of the cache's {heads}")
    if tables.shape[0] != requests or starts.shape[0] != requests + 1:
        raise ValueError(f"tables and starts must be of {requests} requests")
    if tables.shape[1] * cache.block > 2 ** 30:
        raise ValueError("block tables reach 2^30 tokens a request at most")
    _check_devices(cache.k_codes, q, tables, lens, starts)
    group, state = q_heads // heads, _native.gpu(q)
    sizes = (ctypes.c_int64 * 2)()
    library().wq8_kv_attention_workspace(tokens, requests, heads, group, head_dim, state.cus, sizes)
    return ((ctypes.c_longlong * 4)(q.stride(0), q.stride(1), q_heads * head_dim, head_dim), tables.stride(0),
            (tokens, requests, heads, group, head_dim, cache.block, cache.pages), head_dim ** -0.5, DTYPES[q.dtype], state.cus, sizes[0])
