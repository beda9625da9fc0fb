"""Rotary positions with one or several axes on MI355X: the queries and keys of one projection rotated in one launch.

Channels come in pairs (a, b) that turn by the angle position * frequency,

    a' = a cos - b sin,   b' = a sin + b cos,

where every pair belongs to one of up to three axes (time, height, width) and takes that axis's position. Turning back
(inverse=True) is the transpose: it is also the gradient of a rotation with respect to its input.
"""
import ctypes
import math

import torch

from . import DTYPES, _native, library

STYLES = {"pairs": 0, "halves": 1}
MAX_AXES, MAX_TENSORS = 3, 4


class Layouts(dict):
    """Shapes, strides and types that calls have been checked for, and what the kernels are told of them: a decode step's host time is its
    checks (10 us of 19 in rotary()), and its shapes repeat."""
    MOST = 4096

    def keep(self, key, value):
        if len(self) >= self.MOST:
            self.clear()
        self[key] = value
        return value


def _arctan_inverse(x, bits):
    """arctan(1 / x) in parts of 2^-bits, by its series."""
    power = total = (1 << bits) // x
    n = 1
    while power:
        power, n = -power // (x * x), n + 2
        total += power // n
    return total


# 2 pi in parts of 2^-1280 (Machin's formula): a frequency of up to 2^1024 leaves more than the 64 bits of a turn that are kept
_TWO_PI_BITS = 1280
_TWO_PI = 2 * (16 * _arctan_inverse(5, _TWO_PI_BITS) - 4 * _arctan_inverse(239, _TWO_PI_BITS))


def _turn(frequency):
    """frequency / 2 pi modulo one, as the nearest fraction of 2^64 in two's complement: a position times it wraps at whole turns."""
    a, b = frequency.as_integer_ratio()
    whole = b * _TWO_PI
    turns = ((a << _TWO_PI_BITS + 65) + whole) // (2 * whole)
    return (turns + 2 ** 63) % 2 ** 64 - 2 ** 63


class RotaryPlan:
    """Which pairs turn, about which axis and how fast, on one GPU (rotary_plan()). Made once per model."""
    __slots__ = ("sections", "style", "pairs", "turns", "axis", "layouts")

    def __init__(self, sections, style, turns, axis):
        self.sections, self.style, self.pairs, self.turns, self.axis = sections, style, sum(sections), turns, axis
        self.layouts = Layouts()


def rotary_plan(sections, ladder="axis", style="pairs", base=10000.0, frequencies=None, device="cuda"):
    """A plan of sum(sections) rotated pairs a head, sections[a] of them on axis a, in that order.

    ladder 'axis': pair i of a section of n turns by base ** (-i / n) a position, each axis with a ladder of its own; 'joint':
    pair i of all n by base ** (-i / n), one ladder cut into the sections. frequencies (one a pair) replaces both. Frequencies are FP64
    numbers: one of a ladder is within about 2^-53 of itself.
    style 'pairs': pair i is channels 2 i and 2 i + 1; 'halves': channels i and i + sum(sections). Channels past the
    rotated ones pass through."""
    sections = tuple(int(s) for s in sections)
    pairs = sum(sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 1:
        raise ValueError(f"rotary sections must be 1 to {MAX_AXES} positive pair counts, not {sections}")
    if style not in STYLES:
        raise ValueError(f"unknown rotary style {style!r}")
    if frequencies is not None:
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != pairs or not all(map(math.isfinite, frequencies)):
            raise ValueError(f"{pairs} finite rotary frequencies are wanted, one a pair")
    else:
        if ladder not in ("axis", "joint"):
            raise ValueError(f"unknown rotary ladder {ladder!r}")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("the rotary base must be positive and finite")
        steps = [i / n for n in sections for i in range(n)] if ladder == "axis" else [i / pairs for i in range(pairs)]
        frequencies = [float(base) ** -s for s in steps]
    turns = [_turn(f) for f in frequencies]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    packed = torch.tensor(turns + axis, dtype=torch.int64).to(device)  # one copy
    return RotaryPlan(sections, style, packed[:pairs], packed[pairs:].to(torch.int32))


def _check_rows(x, name):
    """(token, head, channel) rows with unit channel stride, 16-byte aligned, heads of a multiple of 8 channels."""
    if x.dim() != 3 or (x.shape[2] > 1 and x.stride(2) != 1):
        raise ValueError(f"{name} must be (tokens, heads, channels) with unit channel stride")
    if x.dtype not in DTYPES:
        raise ValueError(f"{name} must be FP16, BF16 or FP32, not {x.dtype}")
    if x.shape[2] % 8:
        raise ValueError(f"{name} must have heads of a multiple of 8 channels, not {x.shape[2]}")
    size = x.element_size()
    if (x.data_ptr() % 16 or (x.shape[0] > 1 and x.stride(0) * size % 16) or (x.shape[1] > 1 and x.stride(1) * size % 16)):
        raise ValueError(f"rows of {name} must be 16-byte aligned")


def _check_written(x, name):
    """Rows with places of their own, as different workgroups write them."""
    if x.stride(0) >= x.shape[1] * x.stride(1) and x.stride(1) >= x.shape[2]:
        return
    span = 1
    for stride, size in sorted((stride, size) for stride, size in zip(x.stride(), x.shape) if size > 1):
        if stride < span and x.numel():
            raise ValueError(f"rows of {name} must not overlap")
        span += stride * (size - 1)


def _check_devices(*tensors):
    """Tensors on one GPU: the kernels take raw pointers."""
    device = tensors[0].get_device()
    if device < 0:
        raise ValueError("tensors must be on the GPU")
    if any(t.get_device() != device for t in tensors):
        raise ValueError("tensors must be on one GPU")


def _check_aligned(pointers):
    for p in pointers:
        if p & 15:
            raise ValueError("rows must be 16-byte aligned")


def _check_rotary(tensors, positions, plan):
    """What the kernel is told of a call's inputs: tokens, head width, strides of positions, and per tensor heads and strides."""
    if not 1 <= len(tensors) <= MAX_TENSORS:
        raise ValueError(f"rotary takes 1 to {MAX_TENSORS} tensors")
    first = tensors[0]
    for x in tensors:
        _check_rows(x, "rotary rows")
        if x.dtype != first.dtype or x.shape[0] != first.shape[0] or x.shape[2] != first.shape[2]:
            raise ValueError("rotary tensors must agree in type, tokens and head width")
    tokens, _, head_dim = first.shape
    axes = len(plan.sections)
    if 2 * plan.pairs > head_dim:
        raise ValueError(f"the plan turns {2 * plan.pairs} channels, the heads have {head_dim}")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((tokens, axes), (tokens,) if axes == 1 else (tokens, axes)):
        raise ValueError(f"rotary positions must be ({tokens}, {axes}) int32 or int64, not {tuple(positions.shape)} {positions.dtype}")
    _check_devices(*tensors, positions, plan.turns)
    count = len(tensors)
    # a new output is contiguous
    strides = [v for x in tensors for v in (x.shape[1], x.stride(0), x.stride(1), x.shape[1] * head_dim, head_dim)]
    return (ctypes.c_void_p * count, (ctypes.c_longlong * (5 * count))(*strides), positions.stride(0), positions.stride(1) if positions.dim() == 2 else 0,
            positions.dtype == torch.int64, tokens, head_dim, DTYPES[first.dtype])


def rotary(xs, positions, plan, inverse=False, out=None):
    """Rows (tokens, heads, head_dim) of BF16, FP16 or FP32 turned by their positions: a tensor, or a tuple of up to four of one
    type, token count and head width (queries and keys; views of a packed projection). positions: (tokens, axes) int32 or
    int64, or (tokens,) with one axis. inverse turns back. Angles are reduced to parts of a turn as 64-bit integers: that of position
    p is within |p| 2^-65 turns of p times the pair's FP64 frequency. out: tensors of the same shapes whose rows do not overlap, which
    may be the inputs themselves and share memory with them in no other way. Not recorded for autograd: the caller's backward is this
    function with inverse turned over."""
    many = not isinstance(xs, torch.Tensor)
    tensors = tuple(xs) if many else (xs,)
    key = (positions.shape, positions.stride(), positions.dtype, positions.get_device(), *[(x.shape, x.stride(), x.dtype, x.get_device()) for x in tensors])
    layout = plan.layouts.get(key) or plan.layouts.keep(key, _check_rotary(tensors, positions, plan))
    pointers, strides, pos_token, pos_axis, wide, tokens, head_dim, dtype = layout
    if out is None:
        outs = tuple([torch.empty_like(x, memory_format=torch.contiguous_format) for x in tensors])
    else:
        outs = tuple(out) if many else (out,)
        if len(outs) != len(tensors) or any(y.shape != x.shape or y.dtype != x.dtype for x, y in zip(tensors, outs)):
            raise ValueError("rotary outputs do not match its inputs")
        for y in outs:
            _check_rows(y, "rotary outputs")
            _check_written(y, "rotary outputs")
        _check_devices(positions, *outs)
        strides = type(strides)(*[v for x, y in zip(tensors, outs) for v in (x.shape[1], x.stride(0), x.stride(1), y.stride(0), y.stride(1))])
    places, to = [x.data_ptr() for x in tensors], [y.data_ptr() for y in outs]
    _check_aligned(places)
    count = len(places)
    library().call("wq8_rotary", pointers(*places), pointers(*to), strides, count, positions.data_ptr(), pos_token, pos_axis, wide, tokens, plan.turns.data_ptr(),
                   plan.axis.data_ptr(), plan.pairs, head_dim, STYLES[plan.style], inverse, dtype, _native.gpu(positions).stream())
    return outs if many else outs[0]
