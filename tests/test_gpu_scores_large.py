"""Scores of rows with finite logits of any size: as masks, as one token's, as all of a row's.

Tolerances are test_gpu_logits.py's.
"""

import pytest
import torch

import cfm_b200  # noqa: F401
from test_gpu_logits import check_scores, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", [1e4, 1e7, 1e8, 1e9, 3e9, 1e10, 1e11, 1e12, 1e15, 1e20, 1e25, 1e28, 3e29, 1e31])
def test_scores_beside_a_large_value(dtype, fill):
    for rows, vocabulary, start, end in ((3, 8192, 0, 6000), (260, 8192, 0, 6000), (2, 50257, 0, 40000), (2, 1024, 0, 512),
                                         (5, 70000, 30000, 70000)):
        x = logits(rows, vocabulary, dtype, vocabulary)
        tokens = torch.randint(0, vocabulary, (rows,), device="cuda")
        x[:, start:end] = -fill  # a mask
        check_scores(x, tokens, 20)
        x[:, start:end:7] = -fill / 2
        x[:, start:end:5] = -fill * 2
        check_scores(x, tokens, 5)
        x[:, :] = -fill
        check_scores(x, tokens, 5)
        x[:, 77] = fill
        check_scores(x, tokens, 5)
    x = logits(4, 5000, dtype, 3)
    x[:, 100] = fill
    x[1, 4000] = fill
    check_scores(x, torch.tensor([100, 4000, 1, 2], device="cuda"), 20)
    check_scores(x + fill, torch.tensor([100, 4000, 1, 2], device="cuda"), 20)
    check_scores(x - fill, torch.tensor([100, 4000, 1, 2], device="cuda"), 20)
