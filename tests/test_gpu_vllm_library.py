"""The decode study with the library's router and scores: a two-layer model in a child process."""

import json
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def test_two_layer_decode_study_with_the_library_scores():
    pytest.importorskip("vllm")
    env = dict(os.environ, VLLM_LOGGING_LEVEL="WARNING", PYTHONPATH=str(ROOT))
    run = subprocess.run(
        [sys.executable, "-m", "cfm_b200.runtime.vllm_binding", "--layers", "2", "--batch", "4",
         "--prompt-tokens", "64", "--decode-tokens", "8", "--memory-fraction", "0.2", "--library"],
        cwd=ROOT, env=env, capture_output=True, text=True, timeout=900,
    )
    assert run.returncode == 0, run.stderr[-3000:]
    report = json.loads([line for line in run.stdout.splitlines() if line.startswith("{")][-1])
    assert report["decode_steps"] == 7 and report["sparse_rows_per_layer"] == 4 * 7
    assert report["prefill_step_kl"] == 0.0  # the same logits in both runs
    assert 0.0 <= report["kl_stock_to_sparse_mean"] < 0.05
    # Random weights: nearly all of the vocabulary is in play.
    assert 0.0 < report["stock_entropy_mean"] <= math.log(151936)
    assert -math.log(151936) < report["sparse_logprob_of_stock_token_mean"] < 0.0
