"""The speculative decoding example runs the operators together and emits what the model would; a step can be captured."""

from __future__ import annotations

import runpy
import sys
from pathlib import Path

import pytest
import torch

from tklab.kernels.flash_attention import check_device_status
from tklab.kernels.rotary import rotary, rotary_tables
from tklab.kernels.speculative import commit_draft, verify_draft
from tklab.kernels.tree_attention import tree_attention

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


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("batch", "nodes", "capacity"), [(1, 1, 40), (3, 6, 900), (2, 80, 3000)])
def test_a_step_in_a_graph(batch: int, nodes: int, capacity: int) -> None:
    """Rotary, attention, verification and commit captured as one graph: replayed on new data, the bits of the calls."""
    gen = torch.Generator(device="cuda").manual_seed(nodes)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").bfloat16()  # noqa: E731
    cos, sin = rotary_tables(capacity + nodes, 64, device="cuda")
    parents = (torch.arange(nodes, device="cuda") - 1).div(2, rounding_mode="floor").int()
    x = {
        "q": rand(batch, 8, nodes, 64), "k": rand(batch, 2, nodes, 64), "v": rand(batch, 2, nodes, 64),
        "k_cache": rand(batch, 2, capacity, 64), "v_cache": rand(batch, 2, capacity, 64),
        "lens": torch.full((batch,), capacity // 2, dtype=torch.int32, device="cuda"),
        "tokens": torch.randint(0, 50, (batch, nodes), generator=gen, device="cuda"),
    }

    def refill():
        for name in ("q", "k", "v", "k_cache", "v_cache"):
            x[name].copy_(rand(*x[name].shape))
        x["lens"].copy_(torch.randint(0, capacity - nodes, (batch,), generator=gen, device="cuda"))
        x["tokens"].random_(0, 50, generator=gen)
        more["target"].copy_((2.0 * torch.randn(batch, nodes, 50, generator=gen, device="cuda")).softmax(-1))
        more["uniforms"].uniform_(generator=gen)
        more["noise"].exponential_(generator=gen)

    more = {"target": torch.empty(batch, nodes, 50, device="cuda"), "uniforms": torch.empty(batch, nodes, device="cuda"),
            "noise": torch.empty(batch, 50, device="cuda")}

    def step():
        positions = x["lens"][:, None] + torch.arange(nodes, device="cuda")
        q, k = rotary(x["q"], x["k"], cos, sin, positions=positions)
        o = tree_attention(q, x["k_cache"], x["v_cache"], k, x["v"], x["lens"], parents)
        found = verify_draft(more["target"], x["tokens"], more["uniforms"], more["noise"], parents=parents)
        lens = commit_draft(x["k_cache"], x["v_cache"], k, x["v"], found.path, found.path_lens, x["lens"])
        return [o, *found, lens]

    refill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        refill()
        caches = [x[n].clone() for n in ("k_cache", "v_cache")]
        graph.replay()
        got = [t.clone() for t in (*out, x["k_cache"], x["v_cache"])]
        for n, t in zip(("k_cache", "v_cache"), caches, strict=True):
            x[n].copy_(t)
        for a, b in zip(got, [*step(), x["k_cache"], x["v_cache"]], strict=True):
            assert torch.equal(a, b)
    check_device_status()
