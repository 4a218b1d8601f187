"""Speculative decoding of a batch with the framework's operators.

A small decoder with random weights generates for prompts of different
lengths.  Its drafts come from a model of its own embedding and output
weights without the layers between them.  Per step and layer: ``rotary`` places
the drafted tokens' queries and keys at their depths, ``tree_attention``
attends cache and tree; then ``verify_draft`` walks the tree and draws the next
token and ``commit_draft`` writes the accepted rows of all layers.  Prompts
enter the cache as chains through the same operators.  Nothing of a step is
read by the host, which may run ahead of the GPU.

    python examples/speculative_decode.py                     # greedy, a tree of drafts
    python examples/speculative_decode.py --temperature 0.8   # sampled
    python examples/speculative_decode.py --temperature 0.8 --chain 4   # sampled chain, against the draft's probabilities
    python examples/speculative_decode.py --check             # greedy, and compared with the whole sequences in float32
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "triton-kernel-lab_b200"))

from tklab.kernels.flash_attention import check_device_status  # noqa: E402
from tklab.kernels.rotary import rotary, rotary_tables  # noqa: E402
from tklab.kernels.speculative import commit_draft, verify_draft  # noqa: E402
from tklab.kernels.tree_attention import MAX_TREE_NODES, tree_attention  # noqa: E402

VOCAB, LAYERS, Q_HEADS, KV_HEADS, DIM = 1000, 4, 8, 2, 64
HIDDEN = Q_HEADS * DIM
# (node, how many of its likeliest successors are drafted): 11 nodes, the last known token's among them, 4 deep.
CHILDREN = ((0, 3), (1, 2), (2, 1), (4, 2), (5, 1), (7, 1))


def tree_of(children):
    """Parents and depths."""
    parents, depths = [-1], [0]
    for node, count in children:
        parents += [node] * count
        depths += [depths[node] + 1] * count
    return parents, depths


def norm(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.rms_norm(x, (x.shape[-1],))


class Decoder:
    """Pre-norm decoder layers with grouped queries and rotary positions."""

    def __init__(self, capacity: int, seed: int = 0) -> None:
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols, scale=1.0):
            return (torch.randn(rows, cols, generator=gen, device="cuda") * scale * rows**-0.5).bfloat16()

        self.embed = weight(VOCAB, HIDDEN, VOCAB**0.5)
        self.head = weight(HIDDEN, VOCAB, 4.0)
        self.qkv = [weight(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * DIM) for _ in range(LAYERS)]
        self.out = [weight(HIDDEN, HIDDEN, 0.3) for _ in range(LAYERS)]
        self.up = [weight(HIDDEN, 2 * HIDDEN) for _ in range(LAYERS)]
        self.down = [weight(2 * HIDDEN, HIDDEN, 0.3) for _ in range(LAYERS)]
        self.cos, self.sin = rotary_tables(capacity + MAX_TREE_NODES, DIM, device="cuda")

    def logits(self, tokens: torch.Tensor, positions: torch.Tensor, attend) -> torch.Tensor:
        """``attend(layer, q, k, v)`` is the attention of rotated (batch, heads, tokens, DIM) queries and keys."""
        x = self.embed[tokens]
        batch, count = tokens.shape
        for layer in range(LAYERS):
            heads = (norm(x) @ self.qkv[layer]).view(batch, count, -1, DIM).transpose(1, 2)
            q, k, v = heads.split((Q_HEADS, KV_HEADS, KV_HEADS), 1)
            q, k = rotary(q, k, self.cos, self.sin, positions=positions)
            o = attend(layer, q, k, v)
            x = x + o.transpose(1, 2).reshape(batch, count, HIDDEN) @ self.out[layer]
            x = x + torch.nn.functional.gelu(norm(x) @ self.up[layer]) @ self.down[layer]
        return norm(x).float() @ self.head.float()

    def draft_logits(self, tokens: torch.Tensor) -> torch.Tensor:
        return norm(self.embed[tokens]).float() @ self.head.float()

    def full_logits(self, tokens: torch.Tensor) -> torch.Tensor:
        """One sequence at once in plain float32."""
        x = self.embed[tokens].float()
        count = len(tokens)
        cos, sin = self.cos[:count], self.sin[:count]

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        for layer in range(LAYERS):
            heads = (norm(x) @ self.qkv[layer].float()).view(count, -1, DIM).transpose(0, 1)
            q, k, v = heads.split((Q_HEADS, KV_HEADS, KV_HEADS), 0)
            k, v = (t.repeat_interleave(Q_HEADS // KV_HEADS, 0) for t in (turn(k), v))
            scores = (turn(q) @ k.transpose(1, 2)) * DIM**-0.5
            scores.masked_fill_(torch.ones(count, count, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
            x = x + (scores.softmax(-1) @ v).transpose(0, 1).reshape(count, HIDDEN) @ self.out[layer].float()
            x = x + torch.nn.functional.gelu(norm(x) @ self.up[layer].float()) @ self.down[layer].float()
        return norm(x) @ self.head.float()


class Cache:
    """Keys and values of every layer, with each sequence's length."""

    def __init__(self, batch: int, capacity: int) -> None:
        self.k = torch.empty(LAYERS, batch, KV_HEADS, capacity, DIM, dtype=torch.bfloat16, device="cuda")
        self.v = torch.empty_like(self.k)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def run(self, model, tokens, depths, parents, sizes=None):
        """The model on a tree of tokens behind the cache: its logits, and the tree's own keys and values."""
        batch, nodes = tokens.shape
        k_tree = torch.empty(LAYERS, batch, KV_HEADS, nodes, DIM, dtype=torch.bfloat16, device="cuda")
        v_tree = torch.empty_like(k_tree)

        def attend(layer, q, k, v):
            k_tree[layer], v_tree[layer] = k, v
            return tree_attention(
                q, self.k[layer], self.v[layer], k_tree[layer], v_tree[layer], self.lens, parents, tree_sizes=sizes
            )

        return model.logits(tokens, self.lens[:, None] + depths, attend), k_tree, v_tree

    def commit(self, k_tree, v_tree, path, path_lens):
        self.lens = commit_draft(self.k, self.v, k_tree, v_tree, path, path_lens, self.lens)


def prefill(model: Decoder, cache: Cache, prompts: torch.Tensor, lens: torch.Tensor) -> None:
    """The prompts' tokens but the last, in chains of up to ``MAX_TREE_NODES``."""
    for start in range(0, prompts.shape[1] - 1, MAX_TREE_NODES):
        tokens = prompts[:, start : min(start + MAX_TREE_NODES, prompts.shape[1] - 1)]
        chain = torch.arange(tokens.shape[1], dtype=torch.int32, device="cuda")
        sizes = (lens - 1 - start).clamp(0, tokens.shape[1]).int()
        _, k, v = cache.run(model, tokens, chain, None, sizes)
        cache.commit(k, v, chain.expand(tokens.shape).contiguous(), sizes)


def distribution(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    """Probabilities; all on the likeliest token at temperature 0."""
    if temperature > 0.0:
        return (logits / temperature).softmax(-1)
    return torch.zeros_like(logits).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)


def draft_tree(model: Decoder, last: torch.Tensor) -> torch.Tensor:
    """The draft's likeliest tokens after each node that has children: (batch, nodes)."""
    columns = [last]
    for node, count in CHILDREN:
        columns += model.draft_logits(columns[node]).topk(count, -1).indices.unbind(-1)
    return torch.stack(columns, 1)


def draft_chain(model: Decoder, last: torch.Tensor, count: int, temperature: float):
    """Tokens drawn from the draft one after another, with the distributions they were drawn from."""
    columns, probs = [last], []
    for _ in range(count):
        probs.append(distribution(model.draft_logits(columns[-1]), temperature))
        noise = torch.empty_like(probs[-1]).exponential_()
        columns.append((probs[-1] / noise).argmax(-1))
    return torch.stack(columns, 1), torch.stack(probs, 1)


def generate(model, prompts, lens, steps, temperature=0.0, chain=0):
    """``steps`` steps on right-padded prompts: each sequence's tokens, prompt included, and the tokens per step."""
    batch = len(lens)
    parents, depths = tree_of(CHILDREN)
    nodes = chain + 1 if chain else len(parents)
    parents = None if chain else torch.tensor(parents, dtype=torch.int32, device="cuda")
    depths = torch.tensor(range(nodes) if chain else depths, dtype=torch.int32, device="cuda")
    cache = Cache(batch, prompts.shape[1] + steps * nodes)
    prefill(model, cache, prompts, lens)
    last = prompts.gather(1, lens[:, None] - 1)[:, 0]
    found = []
    for _ in range(steps):
        if chain:
            tokens, draft_probs = draft_chain(model, last, chain, temperature)
        else:
            tokens, draft_probs = draft_tree(model, last), None
        logits, k, v = cache.run(model, tokens, depths, parents)
        uniforms = torch.rand(batch, nodes, device="cuda")
        noise = torch.empty(batch, VOCAB, device="cuda").exponential_()
        step = verify_draft(distribution(logits, temperature), tokens, uniforms, noise, parents=parents, draft_probs=draft_probs)
        cache.commit(k, v, step.path, step.path_lens)
        accepted = tokens.gather(1, step.path.clamp_min(0).long())
        last = step.next_tokens
        found.append((accepted, step.path_lens, last))
    check_device_status()
    sequences = [prompts[b, : lens[b]].tolist() for b in range(batch)]
    for accepted, path_lens, token in ((a.tolist(), n.tolist(), t.tolist()) for a, n, t in found):
        for b, sequence in enumerate(sequences):
            sequence += accepted[b][1 : path_lens[b]] + [token[b]]  # node 0 was known
    assert cache.lens.tolist() == [len(s) - 1 for s in sequences]
    return sequences, (sum(map(len, sequences)) - int(lens.sum())) / (steps * batch)


def greedy_gap(model, sequences, lens) -> float:
    """How far below the best a chosen token's logit is at most, in standard deviations of its row's logits."""
    worst = 0.0
    for sequence, first in zip(sequences, lens.tolist(), strict=True):
        tokens = torch.tensor(sequence, device="cuda")
        rows = model.full_logits(tokens)[first - 1 : -1]
        chosen = rows.gather(1, tokens[first:, None])[:, 0]
        worst = max(worst, float(((rows.amax(1) - chosen) / rows.std(1)).max()))
    return worst


def main(argv: list[str] | None = None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--batch", type=int, default=8)
    parser.add_argument("--prompt", type=int, default=300, help="longest prompt")
    parser.add_argument("--steps", type=int, default=32)
    parser.add_argument("--temperature", type=float, default=0.0)
    parser.add_argument("--chain", type=int, default=0, help="draft a chain of so many tokens in place of a tree")
    parser.add_argument("--check", action="store_true", help="compare greedy tokens with whole sequences in float32")
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    lens = torch.randint(1, args.prompt + 1, (args.batch,), device="cuda")
    prompts = torch.randint(0, VOCAB, (args.batch, args.prompt), device="cuda")
    nodes = args.chain + 1 if args.chain else len(tree_of(CHILDREN)[0])
    model = Decoder(args.prompt + args.steps * nodes)
    generate(model, prompts, lens, 1, args.temperature, args.chain)  # first calls load kernels
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    sequences, per_step = generate(model, prompts, lens, args.steps, args.temperature, args.chain)
    end.record()
    torch.cuda.synchronize()
    result = {"tokens_per_step": per_step, "ms": start.elapsed_time(end)}
    if args.check and args.temperature == 0.0:
        result["greedy_gap"] = greedy_gap(model, sequences, lens)
    print(", ".join(f"{name} {value:.3g}" for name, value in result.items()))
    return result


if __name__ == "__main__":
    main()
