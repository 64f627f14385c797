"""Rows of logits as the CUDA library takes them, and calls on their device's current stream."""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _native

TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def check_rows(logits: Tensor, what: str, most_columns: int) -> None:
    """Raise ValueError unless `logits` is a CUDA matrix of contiguous BF16, FP16 or FP32 rows."""
    if (
        logits.ndim != 2
        or logits.dtype not in TYPE_CODES
        or not logits.is_cuda
        or not 1 <= logits.shape[1] <= most_columns
        or logits.shape[0] > 2**28
    ):
        raise ValueError(
            f"{what} must be a CUDA tensor [rows, columns] of BF16, FP16 or FP32 with 1 to "
            f"{most_columns} columns")
    if (logits.shape[1] > 1 and logits.stride(1) != 1) or (
            logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]):
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires grad: this operator has no backward pass")


def rows_struct(logits: Tensor) -> _native.Rows:
    return _native.Rows(logits.data_ptr(), logits.stride(0), logits.shape[0], logits.shape[1],
                        TYPE_CODES[logits.dtype])


def enqueue(name: str, device: torch.device, *arguments: object) -> None:
    """Call an entry point of the library with the current stream of `device` at the end."""
    function = getattr(_native.load(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        code = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _native.check(code, name)


def byref(rows: _native.Rows):
    return ctypes.byref(rows)
