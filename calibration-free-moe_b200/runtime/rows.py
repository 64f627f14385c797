"""Rows of logits as the CUDA library takes them, and calls on their device's current stream."""

from __future__ import annotations

import ctypes
from functools import cache

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _native

TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def wants_gradient(tensor: Tensor) -> bool:
    """Whether autograd would follow an operation on it, backward or forward."""
    return (tensor.requires_grad and torch.is_grad_enabled()) or (
        forward_ad._current_level >= 0 and forward_ad.unpack_dual(tensor).tangent is not None
    )


def check_rows(logits: Tensor, what: str, most_columns: int) -> tuple[_native.Rows, int]:
    """The rows as a structure, and their number; ValueError unless `logits` is a CUDA matrix of
    contiguous BF16, FP16 or FP32 rows."""
    shape = logits.shape
    code = TYPE_CODES.get(logits.dtype)
    if code is None or len(shape) != 2 or not logits.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor [rows, columns] of BF16, FP16 or FP32")
    rows, columns = shape
    if not 1 <= columns <= most_columns or rows > 2**26:
        raise ValueError(f"{what} must have 1 to {most_columns} columns and at most 2^26 rows")
    step, one = logits.stride()
    if (one != 1 and columns > 1) or (step < columns and rows > 1):
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    if wants_gradient(logits):
        raise ValueError(f"{what} requires grad: this operator has no derivative")
    return _native.Rows(logits.data_ptr(), step, rows, columns, code), rows


byref = ctypes.byref


@cache
def entry_point(name: str):
    """A function of the library, which is loaded on first use."""
    return getattr(_native.load(), name)


def enqueue(name: str, index: int, *arguments: object) -> None:
    """Call an entry point with the current stream of device `index` as its last argument."""
    function = entry_point(name)
    if torch.cuda.current_device() == index:
        code = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _native.check(code, name)
