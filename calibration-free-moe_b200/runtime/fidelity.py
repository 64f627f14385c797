"""Scores of next-token logits: what a decode run says of its tokens, and how far two runs are apart.

`vllm_binding.kl_and_top1` states the divergence in torch operations.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from .rows import byref, check_rows, enqueue

MAX_VOCABULARY = 1 << 21
MAX_TOP = 32


class TokenScores(NamedTuple):
    """What `token_logprobs` returns; the last two are None with `top=0`."""

    logprobs: Tensor  # FP32 [T], of the given tokens
    entropy: Tensor  # FP32 [T], nats
    top_ids: Tensor | None  # int32 [T, top], descending
    top_logprobs: Tensor | None  # FP32 [T, top]


def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0) -> TokenScores:
    """Log probability of each row's token, the row's entropy, and its `top` likeliest tokens.

    logits BF16, FP16 or FP32 `[T, V]`, V up to 2^21, rows contiguous and any distance apart (a
    padded vocabulary's slice); T may be zero.  tokens int32 or int64 `[T]`; a token outside of
    the vocabulary has a log probability of NaN.  `top` up to 32; equal logits come by the lowest
    id.  A banned token (-inf) has no probability and a log probability of -inf; a row with NaN or
    +inf, or all of whose tokens are banned, has NaN for all its numbers.  Enqueued on the
    current stream; no gradients.
    """
    struct, rows = check_rows(logits, "Logits", MAX_VOCABULARY)
    index, wide = logits.get_device(), tokens.dtype is torch.int64
    if (
        tokens.shape != (rows,)
        or not (wide or tokens.dtype is torch.int32)
        or not tokens.is_cuda
        or tokens.get_device() != index
        or not tokens.is_contiguous()
    ):
        raise ValueError("Tokens must be contiguous int32 or int64 [rows] on the logits' device")
    if not 0 <= top <= MAX_TOP or top > struct.columns:
        raise ValueError(f"top must be from 0 to {MAX_TOP} and at most the vocabulary's size")
    logprobs = logits.new_empty(rows, dtype=torch.float32)
    entropy = torch.empty_like(logprobs)
    if not top:
        enqueue("cfm_token_logprobs", index, byref(struct), tokens.data_ptr(), wide, 0,
                logprobs.data_ptr(), entropy.data_ptr(), None, None)
        return TokenScores(logprobs, entropy, None, None)
    top_logprobs = logprobs.new_empty((rows, top))
    top_ids = torch.empty_like(top_logprobs, dtype=torch.int32)
    enqueue("cfm_token_logprobs", index, byref(struct), tokens.data_ptr(), wide, top,
            logprobs.data_ptr(), entropy.data_ptr(), top_ids.data_ptr(), top_logprobs.data_ptr())
    return TokenScores(logprobs, entropy, top_ids, top_logprobs)


def compare_logits(reference: Tensor, logits: Tensor) -> tuple[Tensor, Tensor]:
    """KL(softmax(reference) || softmax(logits)) of every pair of rows, and whether their tops agree.

    Both `[T, V]` of one type (BF16, FP16 or FP32), V up to 2^21, each with rows of its own
    distance; T may be zero.  Returns the divergence in nats (FP32 `[T]`) and a bool `[T]`: the
    largest logits of the two rows are at the same token, equal ones by the lowest id.  Rows that
    hardly differ keep their digits: no sums of the size of the logits are subtracted.  The
    divergence is +inf where the reference gives weight to a token that `logits` bans (e^-745 of its
    largest weight at least: not where it masks by a finite value), and NaN where a row has NaN or
    +inf or is banned altogether.  Enqueued on the current stream; no gradients.
    """
    one, _ = check_rows(reference, "Reference logits", MAX_VOCABULARY)
    other, rows = check_rows(logits, "Logits", MAX_VOCABULARY)
    index = logits.get_device()
    if (
        one.rows != rows or one.columns != other.columns or one.type != other.type
        or reference.get_device() != index
    ):
        raise ValueError("Both rows of logits must have one shape, type and device")
    divergence = logits.new_empty(rows, dtype=torch.float32)
    agreement = torch.empty_like(divergence, dtype=torch.bool)
    enqueue("cfm_compare_logits", index, byref(one), byref(other), divergence.data_ptr(),
            agreement.data_ptr())
    return divergence, agreement
