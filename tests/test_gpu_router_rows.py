"""Router rows without a distribution: every weight is NaN, and the ids are in order all the same."""

import math

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200.runtime.routing import route_tokens
from test_gpu_logits import TYPES, logits, ranked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts", [4, 60, 128, 200, 1000])
@pytest.mark.parametrize("renormalize", [True, False])
def test_weights_of_rows_without_a_distribution(dtype, experts, renormalize):
    inf, nan = math.inf, math.nan
    x = logits(9, experts, dtype, experts, 1.5, peak=False)
    x[0, experts - 1] = inf
    x[1, 0] = x[1, 2] = inf
    x[2] = inf
    x[3] = -inf
    x[4, experts // 2] = nan
    x[5] = nan
    x[6, 1], x[6, 3] = nan, inf
    x[7, 1:] = -inf  # one expert has it all
    weights, ids = route_tokens(x, 4, renormalize=renormalize)
    assert torch.equal(ids.long(), ranked(x, 4))
    assert weights[:7].isnan().all()
    assert weights[7].tolist() == [1.0, 0.0, 0.0, 0.0]
    assert weights[8].isfinite().all()
    for more in (route_tokens(x, 4, renormalize=renormalize, weights_dtype=torch.bfloat16)[0],):
        assert more[:7].isnan().all() and not more[7:].isnan().any()
