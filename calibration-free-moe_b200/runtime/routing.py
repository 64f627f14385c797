"""The softmax router in front of the reader and of `RoutedExperts`.

`vllm_binding.route` states the same in torch operations; this is one launch.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .rows import byref, check_rows, enqueue

MAX_EXPERTS = 1024
MAX_TOP_K = 32


def route_tokens(
    logits: Tensor,
    top_k: int,
    *,
    renormalize: bool = True,
    weights_dtype: torch.dtype = torch.float32,
    ids_dtype: torch.dtype = torch.int32,
) -> tuple[Tensor, Tensor]:
    """Router weights and expert ids `[T, K]` of the `top_k` largest of every row of `logits`.

    logits BF16, FP16 or FP32 `[T, E]`, E up to 1024, rows contiguous and any distance apart;
    T may be zero.  The ids (int32 or int64) are in descending order of the logits, equal logits
    by the lowest id, NaN above all.  The weights (FP32 or BF16) are the softmax over all experts
    in FP32, divided by their sum over the picked ones with `renormalize`; a row with NaN or +inf
    or of nothing but -inf has weights of NaN.  What a reader takes as `topk_ids` and
    `topk_weights`.  Enqueued on the current stream; no gradients.
    """
    struct, rows = check_rows(logits, "Router logits", MAX_EXPERTS)
    if not 1 <= top_k <= MAX_TOP_K or top_k > struct.columns:
        raise ValueError(f"top_k must be from 1 to {MAX_TOP_K} and at most the number of experts")
    if weights_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("Router weights are FP32 or BF16")
    if ids_dtype not in (torch.int32, torch.int64):
        raise ValueError("Expert ids are int32 or int64")
    weights = logits.new_empty((rows, top_k), dtype=weights_dtype)
    ids = torch.empty_like(weights, dtype=ids_dtype)
    enqueue("cfm_route_tokens", logits.get_device(), byref(struct), top_k, renormalize,
            ids.data_ptr(), ids_dtype is torch.int64, weights.data_ptr(),
            weights_dtype is torch.bfloat16)
    return weights, ids
