"""A mixture-of-experts layer of INT8 weights for a few tokens.

    routes = route(x, router, 8)                                    # the experts of every token, and their weights
    y = experts(x, routes, gate_up, gate_up_scales, down, down_scales, residual=stream, out=stream)

The experts' weights are the checkpoint's INT8 matrices with FP32 scales per channel, stacked; they are used as stored, and each chosen
expert's are read once for up to 64 of its tokens. Activations are not rotated: weights of a ConvRot checkpoint are not what it takes. Neither call reads anything on the host: a decode step with such layers can be captured.
"""
import ctypes
from typing import NamedTuple

import torch

from . import DTYPES, _check_activation, _native, _row_pitch, library
from ._added import _check_channels, _check_sum
from ._rotary import Layouts, _check_devices

SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_TOP, MAX_CHOICES = 1024, 64, 4096
_route_layouts, _experts_layouts = Layouts(), Layouts()


class Routes(NamedTuple):
    """Which experts each token has, and how they count."""
    ids: torch.Tensor      # (tokens, top) int32
    weights: torch.Tensor  # (tokens, top) float32


def _check_route(x, router, top, score, bias):
    _check_activation(x, aligned=False)
    if x.shape[0] > 1 and x.stride(0) * x.element_size() % 16:
        raise ValueError("activation rows must be 16-byte aligned")
    if router.dim() != 2 or not router.is_contiguous() or router.dtype not in DTYPES or router.shape[1] != x.shape[1]:
        raise ValueError(f"the router must be (experts, {x.shape[1]}) FP16, BF16 or FP32, contiguous")
    count, k = router.shape
    if k < 8 or k % 8 or not 1 <= count <= MAX_EXPERTS:
        raise ValueError(f"a router has 1 to {MAX_EXPERTS} experts over a multiple of 8 channels, not {count} over {k}")
    if not 1 <= top <= min(count, MAX_TOP):
        raise ValueError(f"a token has 1 to {min(count, MAX_TOP)} of the {count} experts, not {top}")
    if score not in SCORES:
        raise ValueError(f"unknown score {score!r}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (count,) or not bias.is_contiguous()):
        raise ValueError(f"the bias must be ({count},) FP32, contiguous")
    if x.shape[0] > 65535 * 16:
        raise ValueError("a route is of 2^20 - 16 tokens at most")
    _check_devices(*[t for t in (x, router, bias) if t is not None])
    sizes = (ctypes.c_int64 * 2)()
    library().wq8_route_workspace(x.shape[0], count, k, sizes)
    return x.shape[0], count, k, _row_pitch(x), DTYPES[x.dtype], DTYPES[router.dtype], sizes[0]


def route(x, router, top, score="softmax", bias=None, normalise=True, factor=1.0):
    """The `top` experts of every row of x (tokens, k) BF16, FP16 or FP32 with 16-byte aligned rows: Routes(ids, weights).

    router: (experts, k) of the same types. The products are FP64 (FP32 sums would leave the choice between near experts to their
    order). score: 'softmax' over all experts or 'sigmoid' of each; bias: (experts,) FP32, added for the choice only. The largest are
    chosen, ties by the lowest index, NaN last, and listed in that order. weights: the chosen scores, with normalise over their sum, times factor."""
    key = (x.shape, x.stride(), x.dtype, x.get_device(), router.shape, router.stride(), router.dtype, router.get_device(), top, score,
           None if bias is None else (bias.shape, bias.stride(), bias.dtype, bias.get_device()))
    tokens, count, k, ldx, dtype, router_dtype, workspace_bytes = _route_layouts.get(key) or _route_layouts.keep(key, _check_route(x, router, top, score, bias))
    x_at, router_at = x.data_ptr(), router.data_ptr()
    if (x_at | router_at) & 15:
        raise ValueError("rows of activations and router must be 16-byte aligned")
    ids = x.new_empty((tokens, top), dtype=torch.int32)
    weights = x.new_empty((tokens, top), dtype=torch.float32)
    logits = x.new_empty(workspace_bytes, dtype=torch.uint8)
    state = _native.gpu(x)
    _native.call_on(library(), state.index, "wq8_route", x_at, ldx, dtype, router_at, router_dtype, _native.ptr(bias), tokens, count, k, top, SCORES[score], normalise, factor,
                   logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), state.stream())
    return Routes(ids, weights)


def _check_codes(codes, scale, shape, name):
    if codes.dtype != torch.int8 or codes.dim() != 3 or not codes.is_contiguous() or codes.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous, 16-byte aligned INT8 of three dimensions")
    if shape is not None and tuple(codes.shape) != shape:
        raise ValueError(f"{name} must be {shape}, not {tuple(codes.shape)}")
    if scale.dtype != torch.float32 or scale.shape != codes.shape[:2] or not scale.is_contiguous():
        raise ValueError(f"scales of {name} must be {tuple(codes.shape[:2])} FP32, contiguous (one a channel)")


def _check_experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual, residual_scale):
    for t in (x, residual):
        if t is None:
            continue
        _check_activation(t, aligned=False)
        if t.dtype == torch.float32 or t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError("experts take FP16 or BF16 rows, and a residual like them")
        if t.shape[0] > 1 and t.stride(0) * 2 % 16:
            raise ValueError("activation rows must be 16-byte aligned")
    if residual_scale is not None:
        if residual is None:
            raise ValueError("a residual_scale belongs to a residual")
        _check_channels(residual_scale, "residual_scale", x)
    _check_codes(gate_up, gate_up_scale, None, "gate_up")
    count, both, k = gate_up.shape
    if k != x.shape[1] or k < 16 or k % 16 or both < 32 or both % 32 or count < 1:
        raise ValueError(f"gate_up must be (experts, 2 hidden, {x.shape[1]}), hidden and channels multiples of 16, not {tuple(gate_up.shape)}")
    _check_codes(down, down_scale, (count, k, both // 2), "down")
    if ids.dtype != torch.int32 or weights.dtype != torch.float32 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or weights.shape != ids.shape:
        raise ValueError("routes must be (tokens, top): ids int32, weights FP32")
    if not (ids.is_contiguous() and weights.is_contiguous()):
        raise ValueError("routes must be contiguous")
    if ids.shape[1] < 1 or ids.numel() > MAX_CHOICES:
        raise ValueError(f"experts() takes at most {MAX_CHOICES} choices (tokens x top) a call, not {tuple(ids.shape)}")
    if both * k >= 2 ** 31 or ((x.shape[0] - 1) * _row_pitch(x) + k) * 2 >= 2 ** 31 or ids.numel() * both * 2 >= 2 ** 31:
        raise ValueError("an expert's matrices, the rows as they lie and the hidden values must each span less than 2 GiB")
    _check_devices(*[t for t in (x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual, residual_scale) if t is not None])
    tokens, top = ids.shape
    sizes = (ctypes.c_int64 * 2)()
    library().wq8_experts_workspace(tokens, top, k, both // 2, sizes)
    return tokens, top, count, k, both // 2, _row_pitch(x), 0 if residual is None else _row_pitch(residual), DTYPES[x.dtype], sizes[0]


def experts(x, routes, gate_up, gate_up_scale, down, down_scale, residual=None, residual_scale=None, out=None):
    """y[t] = sum over j of weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])) with e = ids[t, j], and with a residual
    residual + residual_scale * (...), for the few rows x (tokens, k), BF16 or FP16, 16-byte aligned; at most 4096 choices (tokens x top).

    gate_up: (experts, 2 hidden, k) INT8, the gate's rows first, gate_up_scale: (experts, 2 hidden) FP32; down: (experts, k, hidden),
    down_scale: (experts, k); k and hidden multiples of 16. routes: Routes, or (ids, weights) like them; ids outside the experts are left
    out (a token without any gets zeros, or its residual), and a token may have an expert twice. out: a tensor like x, which may be
    residual or x itself. The activations are used as they are; sums are FP32; the hidden values are held as the sum of two BF16 (17 bits). Not
    recorded for autograd."""
    ids, weights = routes
    key = (x.shape, x.stride(), x.dtype, x.get_device(), ids.shape, ids.stride(), ids.dtype, ids.get_device(), weights.shape, weights.stride(), weights.dtype,
           weights.get_device(), gate_up.shape, gate_up.stride(), gate_up.dtype, gate_up.get_device(), down.shape, down.stride(), down.dtype, down.get_device(),
           gate_up_scale.shape, gate_up_scale.stride(), gate_up_scale.dtype, gate_up_scale.get_device(), down_scale.shape, down_scale.stride(), down_scale.dtype,
           down_scale.get_device(), None if residual is None else (residual.shape, residual.stride(), residual.dtype, residual.get_device()),
           None if residual_scale is None else (residual_scale.shape, residual_scale.stride(), residual_scale.dtype, residual_scale.get_device()))
    layout = _experts_layouts.get(key) or _experts_layouts.keep(key, _check_experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, residual,
                                                                                    residual_scale))
    tokens, top, count, k, hidden, ldx, ldr, dtype, workspace_bytes = layout
    x_at, gate_up_at, down_at, residual_at = x.data_ptr(), gate_up.data_ptr(), down.data_ptr(), _native.ptr(residual)
    if (x_at | gate_up_at | down_at | (residual_at or 0)) & 15:
        raise ValueError("rows of activations and weights must be 16-byte aligned")
    if out is None:
        out, ldo = x.new_empty((tokens, k)), k
    else:
        _check_sum(out, x, x if residual is None else residual)
        ldo = _row_pitch(out)
    workspace = x.new_empty(workspace_bytes, dtype=torch.uint8)
    state = _native.gpu(x)
    _native.call_on(library(), state.index, "wq8_experts", x_at, ldx, dtype, ids.data_ptr(), weights.data_ptr(), gate_up_at, gate_up_scale.data_ptr(), down_at, down_scale.data_ptr(),
                   residual_at, ldr, _native.ptr(residual_scale), out.data_ptr(), ldo, tokens, top, count, k, hidden, workspace.data_ptr(), state.stream())
    return out
