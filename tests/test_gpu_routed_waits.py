"""Waits of the routed experts' tcgen05 kernels that run out: a status, and a context that goes on."""

import ctypes

import pytest
import torch

import device
from cfm_b200 import _native
from cfm_b200.runtime.routed import RoutedExperts
from test_gpu_routed import batch, layer

pytestmark = pytest.mark.gpu


# Passes of 32, 64 and 144 pairs.
@pytest.mark.parametrize("tokens,experts", [(40, 12), (70, 5), (300, 3)])
@pytest.mark.parametrize("hidden,width", [(128, 16), (1152, 272), (2048, 144)])
def test_waits_that_run_out_are_reported(hidden, width, tokens, experts):
    gate_up, down = layer(hidden, width, experts)
    x, ids, weights = batch(tokens, hidden, experts, 2)
    run = RoutedExperts(gate_up, down, 2, tokens)
    want = run(x, ids, weights)
    run.check_status()

    forward = device._load("impatient_experts.cu", _native.nvcc(), *_native.NVCC_FLAGS).cfm_experts_forward
    forward.restype, forward.argtypes = _native.load().cfm_experts_forward.restype, _native.load().cfm_experts_forward.argtypes
    out = torch.empty_like(x)
    call = _native.Call(tokens, 0, 0, 0, 0, 0, x.data_ptr(), ids.data_ptr(), weights.data_ptr(), None, out.data_ptr())
    gave_up = 0
    for _ in range(8):
        run.workspace.status.zero_()
        code = forward(run._layer_ref, run._pointer, tokens, ctypes.byref(call),
                       torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert code == 0
        if int(run.workspace.status):
            gave_up += 1
        else:
            assert torch.equal(out, want)
    assert gave_up
    run.workspace.status.fill_(1)
    with pytest.raises(RuntimeError, match="device-side"):
        run.check_status()

    run.workspace.status.zero_()
    assert torch.equal(run(x, ids, weights), want)
    run.check_status()
