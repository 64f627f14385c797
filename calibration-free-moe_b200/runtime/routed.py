"""The routed experts of a layer as a whole: every channel, for rows that do not take the sparse reader.

`ProgressiveReader` reads the channels that it keeps; `RoutedExperts` reads all of them, from the
same tensors and with the same call, for one token to thousands.  It is the stock side of
`ProgressiveExperts` without an engine (`RoutedExperts.rows`), which `experts.dense_routed_experts` is in
torch operations, and the run that a sparse one is held against.  `ops.register_reader` takes one as it
takes a reader.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _native
from ..activation import ACTIVATION_CODES, GatedActivation
from .rows import wants_gradient


class RoutedWorkspace:
    """Scratch of `RoutedExperts` for up to `capacity` tokens per call.

    One device allocation.  Layers of identical dimensions that run one after another on one
    stream may share it, captured or not; two calls at once may not.
    """

    def __init__(self, hidden_size: int, expert_width: int, experts: int, top_k: int,
                 capacity: int, device: torch.device | str) -> None:
        self.key = (hidden_size, expert_width, experts, top_k)
        self.capacity = capacity
        layer = _native.Experts(hidden_size, expert_width, experts, top_k)
        self.bytes = _native.load().cfm_experts_workspace_bytes(ctypes.byref(layer), capacity)
        if self.bytes < 0:
            raise ValueError(_native.load().cfm_error_string(self.bytes).decode())
        self.buffer = torch.empty(self.bytes, device=device, dtype=torch.uint8)
        self.status = self.buffer[:4].view(torch.int32).zero_()


class RoutedExperts:
    """All channels of the routed experts of one MoE layer.

    gate_up BF16 `[E, 2I, H]` (gate rows, then up rows), contiguous; down BF16, logical `[E, H, I]`
    in the storage of `channel_major_down`: what `ProgressiveReader` takes, and the two may share
    them.  H a multiple of 128, I of 16, E up to 4096, top_k up to 32.  Calls take up to
    `max_tokens` tokens.  Inference only.
    """

    def __init__(
        self,
        gate_up: Tensor,
        down: Tensor,
        top_k: int,
        max_tokens: int,
        *,
        activation: GatedActivation = "silu",
        workspace: RoutedWorkspace | None = None,
    ) -> None:
        if activation not in ACTIVATION_CODES:
            raise ValueError(f"Unknown activation {activation!r}")
        if (
            gate_up.ndim != 3 or gate_up.shape[1] % 2 or gate_up.dtype != torch.bfloat16
            or not gate_up.is_cuda or not gate_up.is_contiguous()
        ):
            raise ValueError("gate_up must be a contiguous CUDA BF16 tensor [E, 2I, H]")
        experts, rows, hidden = gate_up.shape
        width = rows // 2
        if (
            down.shape != (experts, hidden, width) or down.dtype != torch.bfloat16
            or down.device != gate_up.device or not down.transpose(1, 2).is_contiguous()
        ):
            raise ValueError("down must be BF16 [E, H, I] in channel-major storage on gate_up's device")
        if hidden % 128 or width % 16 or not experts or not hidden or not width:
            raise ValueError("Hidden size must be a multiple of 128 and expert width of 16")
        if gate_up.data_ptr() % 16 or down.data_ptr() % 16:
            raise ValueError("Expert weights must start on a 16-byte boundary")
        if workspace is None:
            workspace = RoutedWorkspace(hidden, width, experts, top_k, max_tokens, gate_up.device)
        if (
            workspace.key != (hidden, width, experts, top_k)
            or not 1 <= max_tokens <= workspace.capacity
            or workspace.buffer.device != gate_up.device
        ):
            raise ValueError("Shared workspace must match the layer's dimensions and device")
        self.hidden_size, self.top_k, self.max_tokens = hidden, top_k, max_tokens
        self.gate_up, self.down, self.workspace = gate_up.detach(), down.detach(), workspace
        self._layer = _native.Experts(hidden, width, experts, top_k, ACTIVATION_CODES[activation], 0,
                                      gate_up.data_ptr(), down.data_ptr())
        self._layer_ref = ctypes.byref(self._layer)
        self._pointer = ctypes.c_void_p(workspace.buffer.data_ptr())
        self._forward = _native.load().cfm_experts_forward
        self._device = gate_up.device

    def __call__(
        self,
        hidden: Tensor,
        ids: Tensor,
        weights: Tensor,
        padding: Tensor | None = None,
        out: Tensor | None = None,
    ) -> Tensor:
        """The layer's routed-expert output; arguments and types as `ProgressiveReader.__call__`.

        hidden BF16 `[T, H]`; ids (int32 or int64) and weights (FP32 or BF16) `[T, K]`; padding
        bool `[T]` marks rows that read nothing and produce zeros.  An id outside of the layer's
        experts adds nothing.  Writes `[T, H]` into `out` (allocated if None; it may not overlap the
        other arguments) on the current stream.
        """
        if wants_gradient(hidden) or wants_gradient(weights):
            raise ValueError("Routed input requires grad: this operator has no derivative")
        tokens = hidden.shape[0] if hidden.ndim == 2 else 0
        device = self._device
        if (
            not 1 <= tokens <= self.max_tokens
            or hidden.shape[1] != self.hidden_size
            or hidden.dtype != torch.bfloat16
            or hidden.device != device
            or not hidden.is_contiguous()
            or hidden.data_ptr() % 16
            or ids.shape != (tokens, self.top_k)
            or weights.shape != ids.shape
            or ids.device != device
            or weights.device != device
            or ids.dtype not in (torch.int32, torch.int64)
            or weights.dtype not in (torch.float32, torch.bfloat16)
            or not ids.is_contiguous()
            or not weights.is_contiguous()
            or (
                padding is not None
                and (
                    padding.shape != (tokens,)
                    or padding.device != device
                    or padding.dtype != torch.bool
                    or not padding.is_contiguous()
                )
            )
            or (
                out is not None
                and (
                    out.shape != hidden.shape
                    or out.dtype != hidden.dtype
                    or out.device != device
                    or not out.is_contiguous()
                    or out.data_ptr() % 16
                )
            )
        ):
            raise ValueError("Routed input exceeds the prepared token/expert contract")
        if out is None:
            out = torch.empty_like(hidden)
        call = _native.Call(
            tokens, ids.dtype == torch.int64, weights.dtype == torch.bfloat16, 0, 0, 0,
            hidden.data_ptr(), ids.data_ptr(), weights.data_ptr(),
            padding.data_ptr() if padding is not None else None, out.data_ptr(),
        )
        index = device.index
        if torch.cuda.current_device() == index:
            self._enqueue(call, index)
        else:
            with torch.cuda.device(index):
                self._enqueue(call, index)
        return out

    def _enqueue(self, call: _native.Call, index: int) -> None:
        code = self._forward(self._layer_ref, self._pointer, self.workspace.capacity,
                             ctypes.byref(call), torch._C._cuda_getCurrentRawStream(index))
        if code:
            _native.check(code, "cfm_experts_forward")

    def check_status(self) -> None:
        """Raise if a wait inside a kernel ran out (they end after a second) in a call that used this
        workspace since the last report; the rows of those calls, of any layer that shares it, are
        not to be trusted.  Reporting clears the status.  Waits for the device, whatever the stream."""
        torch.cuda.synchronize(self._device)
        if int(self.workspace.status):
            self.workspace.status.zero_()
            raise RuntimeError("routed-expert kernels reported a device-side error")

    def rows(self, x: Tensor, topk_weights: Tensor, topk_ids: Tensor) -> Tensor:
        """Any number of rows, in calls of at most `max_tokens`: the stock callable of
        `ProgressiveExperts`.  As with its reader, the program calls `check_status` where it
        synchronises anyway; nothing here does."""
        x, ids, weights = x.contiguous(), topk_ids.contiguous(), topk_weights.contiguous()
        out = torch.empty_like(x)
        for start in range(0, x.shape[0], self.max_tokens):
            part = slice(start, start + self.max_tokens)
            self(x[part], ids[part], weights[part], out=out[part])
        return out
