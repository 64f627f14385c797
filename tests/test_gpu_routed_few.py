"""Calls of up to 16 pairs: a token's output bits whatever stands beside it.

Each call's tokens come again alone, in parts and in another order; which experts are busy, how many pairs they have and
whose pairs come first is different every time.
"""

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.runtime.routed import RoutedExperts
from test_gpu_routed import batch, check, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k,tokens", [(1, 16), (1, 9), (2, 8), (3, 5), (4, 4), (5, 3), (6, 2), (8, 2), (16, 1)])
@pytest.mark.parametrize("experts", [2, 4, 9, 64])
@pytest.mark.parametrize("hidden,width", [(256, 80), (1152, 704), (2048, 768)])
def test_bits_of_a_token_in_a_small_call(hidden, width, experts, top_k, tokens):
    gate_up, down = layer(hidden, width, experts)
    run = RoutedExperts(gate_up, down, top_k, 16)
    for seed in range(4):
        x, ids, weights = batch(tokens, hidden, max(experts, top_k), top_k, seed + 1)
        ids = ids % experts  # some tokens have an expert twice
        if seed == 3:
            ids[0, 0] = -1
        out = run(x, ids, weights)
        for order in ([*range(tokens)][::-1], [t for t in range(tokens) if t % 2 == 0], *[[t] for t in range(tokens)]):
            at = torch.tensor(order, device="cuda")
            assert torch.equal(run(x[at], ids[at], weights[at]), out[at])
        padding = torch.arange(tokens, device="cuda") % 3 == 1
        assert torch.equal(run(x, ids, weights, padding)[~padding], out[~padding])


@pytest.mark.parametrize("top_k,tokens", [(1, 16), (2, 8), (3, 5), (4, 4), (8, 2), (16, 1)])
@pytest.mark.parametrize("experts", [1, 2, 5, 40])
def test_definition_of_small_calls(experts, top_k, tokens):
    gate_up, down = layer(512, 208, experts)
    x, ids, weights = batch(tokens, 512, max(experts, top_k), top_k)
    ids = ids % experts
    check(gate_up, down, x, ids, weights)
    padding = torch.arange(tokens, device="cuda") % 3 == 1
    ids[tokens // 2, top_k - 1] = experts
    check(gate_up, down, x, ids.long(), weights.bfloat16(), padding)
