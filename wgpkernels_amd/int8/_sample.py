"""The next tokens of a decode step, drawn on the GPU by given random numbers.

    tokens = sample(logits, torch.rand(len(logits), device="cuda"), temperature=0.7, top_k=50, top_p=0.9)

Nothing is read on the host: a step that ends with it can be captured, and the tokens feed the next one.
"""
import ctypes

import torch

from . import DTYPES, _native, library
from ._rotary import Layouts, _check_devices

MAX_VOCABULARY, MAX_ROWS = 2 ** 24, 2 ** 17
_layouts = Layouts()


def _check_sample(logits, draws, temperature, top_k, top_p, min_p):
    """(rows, vocabulary, row pitch, dtype, workspace bytes, and those of a call that cuts nothing)"""
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1) or logits.dtype not in DTYPES:
        raise ValueError("logits must be (rows, vocabulary) FP16, BF16 or FP32 with unit column stride")
    rows, vocabulary = logits.shape
    if not 1 <= vocabulary <= MAX_VOCABULARY or rows > MAX_ROWS:
        raise ValueError(f"logits must be at most {MAX_ROWS} rows over a vocabulary of 1 to {MAX_VOCABULARY}, not {tuple(logits.shape)}")
    if draws.shape != (rows,) or draws.dtype != torch.float32 or not draws.is_contiguous():
        raise ValueError(f"draws must be ({rows},) FP32, contiguous: a number of [0, 1) a row")
    tensors = []
    for t, dtype, name in ((temperature, torch.float32, "temperature"), (top_k, torch.int32, "top_k"), (top_p, torch.float32, "top_p"),
                           (min_p, torch.float32, "min_p")):
        if isinstance(t, torch.Tensor):
            if t.shape != (rows,) or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be a number, or ({rows},) {str(dtype).removeprefix('torch.')}, contiguous")
            tensors.append(t)
    _check_devices(logits, draws, *tensors)
    sizes = (ctypes.c_int64 * 2)()
    library().wq8_sample_workspace_for(rows, vocabulary, sizes)
    return rows, vocabulary, logits.stride(0) if rows > 1 else vocabulary, DTYPES[logits.dtype], sizes[0], sizes[1]


def _kind(option):
    return (option.shape, option.stride(), option.dtype, option.get_device()) if isinstance(option, torch.Tensor) else None


def _pair(option):
    """(address or None, value) of an option."""
    return (option.data_ptr(), 0) if isinstance(option, torch.Tensor) else (None, option)


def sample(logits, draws, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A token of every row of logits (rows, vocabulary), BF16, FP16 or FP32 with unit column stride: (rows,) int64.

    A token's weight is exp((logit - the row's largest) / temperature), in 64 bits. top_k keeps the k heaviest tokens (0 or below, or
    the vocabulary's size and above: all); of these top_p the fewest, heaviest first, whose weights reach top_p of their sum (1: all; always at least
    one); of these min_p those of at least min_p of the heaviest's weight. Equal logits go by the lowest index. The token drawn is the
    first, in the vocabulary's order, up to which the kept weights pass draws[row] (FP32, in [0, 1)) of their sum. A temperature of 0 (or below) takes
    the first largest logit. Each option is a number, held in FP32, or a (rows,) tensor (FP32, top_k int32).

    Weights are held as whole numbers of units, so that their sums are the same whatever order they are taken in: 2^-44 of the heaviest, in vocabularies
    above 2^18 2^-52 of it or less than 2^-60 of the sum. Those below half a unit are 0. Together a row's weights are off by at most 2^-27 of their sum, less than a
    draw's last bit (2^-24). NaN and -infinity are never drawn; infinities share all weight; a row with nothing else gives -1."""
    key = (logits.shape, logits.stride(), logits.dtype, logits.get_device(), draws.shape, draws.stride(), draws.dtype, draws.get_device(), _kind(temperature),
           _kind(top_k), _kind(top_p), _kind(min_p))
    rows, vocabulary, ld, dtype, workspace_bytes, least_bytes = _layouts.get(key) or _layouts.keep(key, _check_sample(logits, draws, temperature, top_k, top_p, min_p))
    cuts = isinstance(top_k, torch.Tensor) or isinstance(top_p, torch.Tensor) or 0 < top_k < vocabulary or not top_p >= 1
    tokens = draws.new_empty(rows, dtype=torch.int64)
    workspace = draws.new_empty(workspace_bytes if cuts else least_bytes, dtype=torch.uint8)
    state = _native.gpu(logits)
    if not isinstance(top_k, torch.Tensor):
        top_k = max(0, min(top_k, MAX_VOCABULARY))  # the C interface has 32 bits
    _native.call_on(library(), state.index, "wq8_sample", logits.data_ptr(), ld, dtype, draws.data_ptr(), *_pair(temperature), *_pair(top_k), *_pair(top_p),
                    *_pair(min_p), rows, vocabulary, tokens.data_ptr(), workspace.data_ptr(), state.stream())
    return tokens
