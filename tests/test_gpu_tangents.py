"""Forward-mode tangents: the operators of the exact side have no derivative, and say so in either direction."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.func import jvp

import cfm_b200  # noqa: F401
from cfm_b200.runtime.fidelity import compare_logits, token_logprobs
from cfm_b200.runtime.routed import RoutedExperts
from cfm_b200.runtime.routing import route_tokens
from test_gpu_routed import batch, layer

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    logits, tokens = torch.randn((3, 64), device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int64)
    x, ids, weights = batch(3, 256, 4, 2)
    run = RoutedExperts(*layer(256, 48, 4), 2, 8)
    calls = [
        (logits, lambda t: route_tokens(t, 4)), (logits, lambda t: token_logprobs(t, tokens).logprobs),
        (logits, lambda t: compare_logits(t, logits)[0]), (logits, lambda t: compare_logits(logits, t)[0]),
        (x, lambda t: run(t, ids, weights)), (weights, lambda t: run(x, ids, t)),
    ]
    for primal, call in calls:
        with forward_ad.dual_level():
            for context in (torch.enable_grad(), torch.no_grad()):
                with context, pytest.raises(ValueError, match="grad"):
                    call(forward_ad.make_dual(primal, torch.ones_like(primal)))
            call(primal)  # without a tangent
        with pytest.raises(ValueError, match="grad"):
            jvp(call, (primal,), (torch.ones_like(primal),))
