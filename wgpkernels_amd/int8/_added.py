"""The residual's addition, RMS norm and 8-bit preparation of a linear's input in one launch, and what prepared codes stand for.

A linear adds its own branch to the residual stream (residual=). A branch that comes from elsewhere, as a sum over ranks or two branches
side by side, is added here, on the way into the next linear:

    prepared, stream = add_prepare(branch, stream, path="block", act_weight=norm, eps=1e-6, out=stream)
    y = linear_prepared(prepared, weight, scales, bias)
"""
import torch

from . import DTYPES, Prepared, _check_activation, _native, _row_pitch, library
from ._rotary import Layouts, _check_devices

_PATHS = {"block": 0, "exact": 1, "row": 1, "lines": 2, "small": 2}
_layouts = Layouts()


def _check_channels(t, name, x):
    if t.shape != (x.shape[1],) or t.dtype != x.dtype or (t.shape[0] > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be ({x.shape[1]},) of the activations' type, contiguous")


def _check_added(x, residual, residual_scale, group, path, act_weight):
    """Rows, channels and row pitches of a call."""
    for t in (x, residual):
        _check_activation(t, aligned=False)
    if x.dtype == torch.float32 or residual.dtype != x.dtype or residual.shape != x.shape:
        raise ValueError("add_prepare takes two FP16 or two BF16 tensors of one shape")
    if path not in _PATHS:
        raise ValueError(f"unknown INT8 path {path!r}")
    m, k = x.shape
    if k < 8 or k % 8:
        raise ValueError(f"rows must have a multiple of 8 channels, not {k}")
    if m >= 2 ** 24:
        raise ValueError("add_prepare takes fewer than 2^24 rows")
    if group not in (0, 16, 64, 256) or (group and k % group):
        raise ValueError(f"ConvRot groups are of 16, 64 or 256 channels and divide the rows, not {group} of {k}")
    for t in (x, residual):
        if m > 1 and t.stride(0) * 2 % 16:
            raise ValueError("activation rows must be 16-byte aligned")
    for t, name in ((residual_scale, "residual_scale"), (act_weight, "act_weight")):
        if t is not None:
            _check_channels(t, name, x)
    _check_devices(*[t for t in (x, residual, residual_scale, act_weight) if t is not None])
    return m, k, _row_pitch(x), _row_pitch(residual), DTYPES[x.dtype]


def _rows_meet(a, b):
    """Whether rows of a and rows of b (of one width and type) share memory."""
    m, k = a.shape
    if not m:
        return False
    apart, pitch = (a.data_ptr() - b.data_ptr()) // a.element_size(), _row_pitch(a)
    if pitch == _row_pitch(b) and pitch >= k:
        return any(abs(apart - i * pitch) < k for i in (apart // pitch, apart // pitch + 1) if abs(i) < m)
    return -((m - 1) * pitch + k) < apart < (m - 1) * _row_pitch(b) + k


def _check_sum(out, x, residual):
    _check_activation(out)
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("the sum's tensor does not match the activations")
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("rows of the sum must not overlap")
    for t in (x, residual):
        same = t.data_ptr() == out.data_ptr() and _row_pitch(t) == _row_pitch(out)
        if not same and _rows_meet(out, t):
            raise ValueError("the sum may be written over an input in its place, and overlap it in no other way")
    _check_devices(x, out)


def add_prepare(x, residual, residual_scale=None, group=0, path="block", act_weight=None, eps=0.0, out=None):
    """(prepared, sum) of sum = residual + residual_scale * x (x, residual: 2-D BF16 or FP16 rows, 16-byte aligned, of one shape;
    residual_scale: a value a channel in their type, or None), added in FP32 and held in their type; prepared: the sum's
    prepare(sum, group, path, "rms_norm", act_weight, eps), bit for bit. out: the sum's tensor, which may be x or residual itself and
    overlaps them in no other way. One launch, which neither allocates more than the outputs nor waits. Not recorded for autograd."""
    key = (x.shape, x.stride(), x.dtype, x.get_device(), residual.shape, residual.stride(), residual.dtype, residual.get_device(), group, path,
           None if residual_scale is None else (residual_scale.shape, residual_scale.stride(), residual_scale.dtype, residual_scale.get_device()),
           None if act_weight is None else (act_weight.shape, act_weight.stride(), act_weight.dtype, act_weight.get_device()))
    m, k, ldx, ldr, dtype = _layouts.get(key) or _layouts.keep(key, _check_added(x, residual, residual_scale, group, path, act_weight))
    x_at, residual_at, scale_at, weight_at = x.data_ptr(), residual.data_ptr(), _native.ptr(residual_scale), _native.ptr(act_weight)
    if (x_at | residual_at | (scale_at or 0) | (weight_at or 0)) & 15:
        raise ValueError("activation rows and channels must be 16-byte aligned")
    if out is None:
        out, lds = x.new_empty((m, k)), k
    else:
        _check_sum(out, x, residual)
        lds = _row_pitch(out)
    mode = _PATHS[path]
    lo = scale = None
    if mode == 2:
        values = x.new_empty((m, k))
    else:
        values = x.new_empty((m, k), dtype=torch.int8)
        scale = x.new_empty(m if mode else (m, (k + 127) // 128), dtype=torch.float32)
        lo = torch.empty_like(values) if path == "exact" else None
    state = _native.gpu(x)
    _native.call_on(library(), state.index, "wq8_add_prepare", x_at, ldx, residual_at, ldr, scale_at, out.data_ptr(), lds, mode, values.data_ptr(), _native.ptr(lo),
                   _native.ptr(scale), m, k, dtype, group, weight_at, eps, state.stream())
    return Prepared(path, values, lo, scale, x.dtype), out


def prepared_values(prepared):
    """What a preparation stands for, in the activations' type: code * scale, or (hi + lo / 254) * scale, rounded once; the rows
    themselves on the few-token paths."""
    q, lo, scale = prepared.x, prepared.lo, prepared.scale
    if prepared.path in ("lines", "small"):
        return q
    m, k = q.shape
    blocks = prepared.path == "block"
    if k % 8 or scale.numel() != (m * ((k + 127) // 128) if blocks else m) or not all(t is None or t.is_contiguous() for t in (q, lo, scale)):
        raise ValueError("prepared codes must be contiguous rows of a multiple of 8 channels with their scales")
    if q.data_ptr() % 8 or (lo is not None and lo.data_ptr() % 8):
        raise ValueError("prepared codes must be 8-byte aligned")
    _check_devices(q, scale)
    out = torch.empty((m, k), dtype=prepared.dtype, device=q.device)
    state = _native.gpu(q)
    _native.call_on(library(), state.index, "wq8_prepared_values", q.data_ptr(), _native.ptr(lo), scale.data_ptr(), out.data_ptr(), m, k, blocks, DTYPES[prepared.dtype],
                   state.stream())
    return out
