"""The speculative decoding example runs the operators together and emits what the model would."""

from __future__ import annotations

import runpy
import sys
from pathlib import Path

import pytest
import torch

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"
gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU is required")


@pytest.fixture(scope="module")
def example():
    path = list(sys.path)
    found = runpy.run_path(str(EXAMPLE))
    sys.path[:] = path
    return found


def test_tree_is_one(example) -> None:
    parents, depths = example["tree_of"](example["CHILDREN"])
    assert parents[0] == -1 and all(0 <= p < c for c, p in enumerate(parents) if c)
    assert all(depths[c] == depths[p] + 1 for c, p in enumerate(parents) if c)
    assert len(parents) == 11 and max(depths) == 4


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("options", [[], ["--batch", "3", "--prompt", "700", "--steps", "12"], ["--chain", "5"], ["--batch", "1", "--prompt", "1"]])
def test_greedy_tokens_are_the_models(example, options: list[str]) -> None:
    """About 40 roundings to bfloat16 (2^-9 each, in quadrature 1.3 %) lie between a logit and its float32 value; of the
    1000 logits of a row the two compared are off by at most 5 of these together in opposite directions: 10 x 1.3 % of
    the row's spread, doubled."""
    result = example["main"]([*options, "--check"])
    assert result["greedy_gap"] <= 0.26
    assert result["tokens_per_step"] > 1.2  # drafts are accepted


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("options", [[], ["--chain", "4"]])
def test_sampled(example, options: list[str]) -> None:
    result = example["main"]([*options, "--temperature", "0.8"])
    assert 1.0 <= result["tokens_per_step"] <= 5.0
