"""The status of a workspace: reported once, for all layers that share it."""

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.runtime.routed import RoutedExperts, RoutedWorkspace
from test_gpu_routed import batch, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [2, 30])
def test_a_report_clears_the_status(tokens):
    workspace = RoutedWorkspace(256, 48, 4, 2, 32, "cuda")
    runs = [RoutedExperts(*layer(256, 48, 4, seed), 2, 32, workspace=workspace) for seed in (1, 2)]
    x, ids, weights = batch(tokens, 256, 4, 2)
    for run in runs:
        run(x, ids, weights)
        run.check_status()
    workspace.status.fill_(1)  # as a kernel does
    runs[0](x, ids, weights)
    with pytest.raises(RuntimeError, match="device-side"):
        runs[1].check_status()
    for run in runs:
        run.check_status()
        run(x, ids, weights)
        run.check_status()


def test_a_call_on_another_stream_is_waited_for():
    workspace = RoutedWorkspace(256, 48, 4, 2, 32, "cuda")
    run = RoutedExperts(*layer(256, 48, 4), 2, 32, workspace=workspace)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)  # some 25 ms
        workspace.status.fill_(1)
    with pytest.raises(RuntimeError, match="device-side"):
        run.check_status()
    run.check_status()
