"""Speculative decoding around the attention (B200): :func:`verify_draft`
accepts drafted tokens against the target's probabilities and draws the next
one, :func:`commit_draft` writes the accepted tokens' keys and values into
the cache.  Both leave their results on the GPU, so a decoding step needs no
copy to the host.

A step, for drafted trees (``parents``) or chains (``parents=None``)::

    q, k = rotary(q, k, cos, sin, positions=kv_lens[:, None] + depth)
    o = tree_attention(q, k_cache, v_cache, k, v, kv_lens, parents)
    ...                                   # the rest of the model: target_probs
    path, path_lens, token = verify_draft(target_probs, tokens, uniforms, noise, parents=parents)
    kv_lens = commit_draft(k_cache, v_cache, k, v, path, path_lens, kv_lens)
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from tklab._tensors import binding, contiguous, dense, require_cache
from tklab.kernels.flash_attention import _NATIVE_DTYPE, _after_launch
from tklab.kernels.tree_attention import MAX_TREE_NODES, check_lens, check_parents

_PROB_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_TOKEN_TYPES = (torch.int32, torch.int64)


class Verification(NamedTuple):
    """What :func:`verify_draft` found for each sequence of the batch."""

    path: torch.Tensor  # (batch, nodes) int32: the accepted nodes from node 0 on, then -1
    path_lens: torch.Tensor  # (batch,) int32: how many (node 0 counts)
    next_tokens: torch.Tensor  # (batch,), the tokens' dtype


def _prepare_verify(target_probs, tokens, uniforms, noise, parents, draft_probs, tree_sizes) -> tuple:
    """Check the contract; return the arguments with whatever the kernel cannot read in place copied."""
    if target_probs.ndim != 3 or 0 in target_probs.shape:
        raise ValueError("target_probs must be a non-empty (batch, nodes, vocab) tensor")
    batch, nodes, vocab = target_probs.shape
    if nodes > MAX_TREE_NODES:
        raise ValueError(f"verification supports up to {MAX_TREE_NODES} nodes")
    if target_probs.dtype not in _PROB_TYPES:
        raise ValueError("target_probs must be float32, bfloat16 or float16")
    if tokens.shape != (batch, nodes) or tokens.dtype not in _TOKEN_TYPES:
        raise ValueError("tokens must be an int32 or int64 tensor of shape (batch, nodes)")
    if uniforms.shape != (batch, nodes) or uniforms.dtype != torch.float32:
        raise ValueError("uniforms must be a float32 tensor of shape (batch, nodes)")
    if noise.shape != (batch, vocab) or noise.dtype != torch.float32:
        raise ValueError("noise must be a float32 tensor of shape (batch, vocab)")
    if draft_probs is not None:
        if parents is not None:
            raise ValueError("draft_probs are supported for chains only (parents=None)")
        if draft_probs.shape != (batch, nodes - 1, vocab) or draft_probs.dtype != target_probs.dtype:
            raise ValueError("draft_probs must be (batch, nodes - 1, vocab) in the type of target_probs")
    device = target_probs.device
    if not device == tokens.device == uniforms.device == noise.device or (
        draft_probs is not None and draft_probs.device != device
    ):
        raise ValueError("verification needs its tensors on one device")
    if device.type != "cuda":
        raise ValueError("verification requires CUDA tensors")
    check_parents(parents, batch, nodes, device)
    check_lens(tree_sizes, "tree_sizes", batch, device)

    def vocab_contiguous(x: torch.Tensor) -> torch.Tensor:
        return x if x.stride(2) == 1 else x.contiguous()

    return (
        vocab_contiguous(target_probs), tokens.contiguous(), uniforms.contiguous(), noise.contiguous(), contiguous(parents),
        None if draft_probs is None else vocab_contiguous(draft_probs), contiguous(tree_sizes),
    )


def verify_draft(
    target_probs: torch.Tensor,
    tokens: torch.Tensor,
    uniforms: torch.Tensor,
    noise: torch.Tensor,
    *,
    parents: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
    tree_sizes: torch.Tensor | None = None,
) -> Verification:
    """Walk each sequence's drafted tree as far as the target agrees and draw the next token.

    Node 0 is the last known token, node ``c > 0`` a drafted token
    ``tokens[b, c]`` that continues its parent ``n``; ``p = target_probs[b,
    n]`` is the target's distribution after node ``n``.  From node 0 on, a
    node's children are tried in index order:

    * without ``draft_probs`` (the drafts are what they are, e.g. the likeliest
      tokens of a draft model): accepted if ``u (1 - S) < p(x)``, ``S`` the mass
      of the different tokens of its earlier siblings; a token already tried is refused;
    * with ``draft_probs`` (chains only; ``draft_probs[b, n]`` the distribution that
      node ``n + 1`` was drawn from): accepted if ``u q(x) < p(x)``.

    At the last accepted node the next token is ``argmax_v w_v / noise[b,
    v]`` (lowest index of equals), with ``w`` = ``p`` without the tried tokens,
    ``max(p - q, 0)`` with ``draft_probs``, and ``p`` itself at a node without
    children or where ``w`` has nothing left.  With uniform numbers in [0, 1)
    and exponential noise the emitted tokens follow the target's distribution.

    Args:
        target_probs: (batch, nodes, vocab), float32, bfloat16 or float16; 1 to 256 nodes.
        tokens: (batch, nodes) int32 or int64; a token outside the vocabulary is refused.
        uniforms: (batch, nodes) float32 in [0, 1).
        noise: (batch, vocab) float32, positive (``torch.Tensor.exponential_``).
        parents: (batch, nodes) or (nodes,) int32, ``parents[c] < c``; None: a chain.
        draft_probs: (batch, nodes - 1, vocab), the type of ``target_probs``.
        tree_sizes: (batch,) int32, nodes in use (0: no path, next token -1).
    """
    args = (target_probs, tokens, uniforms, noise, parents, draft_probs, tree_sizes)
    found = binding.verify_draft(*args)
    if found is None:
        found = binding.verify_draft(*_prepare_verify(*args))
        if found is None:
            raise ValueError("verification: unsupported arguments")
    _after_launch(target_probs.device)
    return Verification._make(found)


def _prepare_commit(k_cache, v_cache, k_tree, v_tree, path, path_lens, kv_lens) -> tuple:
    """Check the contract; return the arguments with whatever the kernel cannot read in place copied."""
    if not k_cache.ndim == v_cache.ndim == k_tree.ndim == v_tree.ndim or k_cache.ndim not in (4, 5) or (
        k_cache.shape != v_cache.shape or k_tree.shape != v_tree.shape
    ):
        raise ValueError(
            "K and V caches, and the tree's keys and values, must have identical shapes: ([layers,] batch, heads, rows, dim)"
        )
    batch, kv_heads, _, head_dim = k_cache.shape[-4:]
    nodes = k_tree.shape[-2]
    if k_tree.shape != (*k_cache.shape[:-4], batch, kv_heads, nodes, head_dim):
        raise ValueError("the caches and the tree disagree on layers, batch, heads or head_dim")
    if 0 in k_cache.shape or nodes == 0:
        raise ValueError("commit does not support empty dimensions")
    if nodes > MAX_TREE_NODES:
        raise ValueError(f"commit supports up to {MAX_TREE_NODES} nodes")
    if head_dim % 8 or head_dim > 256:
        raise ValueError("commit requires head_dim to be a multiple of 8 up to 256")
    dtype = k_cache.dtype
    if dtype not in _NATIVE_DTYPE or not dtype == v_cache.dtype == k_tree.dtype == v_tree.dtype:
        raise ValueError("caches and tree must share one dtype: float16 or bfloat16")
    device = k_cache.device
    if not device == v_cache.device == k_tree.device == v_tree.device:
        raise ValueError("caches and tree must be on the same device")
    if device.type != "cuda":
        raise ValueError("commit requires CUDA tensors")
    if path.shape != (batch, nodes) or path.dtype != torch.int32 or path.device != device:
        raise ValueError("path must be an int32 tensor of shape (batch, nodes) on the same device")
    check_lens(path_lens, "path_lens", batch, device)
    check_lens(kv_lens, "kv_lens", batch, device)
    require_cache(k_cache, "the K cache")
    require_cache(v_cache, "the V cache")
    return (
        k_cache, v_cache, dense(k_tree), dense(v_tree), path.contiguous(), path_lens.contiguous(), kv_lens.contiguous()
    )


def commit_draft(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    path: torch.Tensor,
    path_lens: torch.Tensor,
    kv_lens: torch.Tensor,
) -> torch.Tensor:
    """Write the accepted rows into the cache, in place, and return the new lengths.

    Row ``path[b, i]`` (``i < path_lens[b]``) of ``k_tree`` and ``v_tree`` goes to
    cache row ``kv_lens[b] + i``.  Caches (batch, kv_heads, seq_kv, head_dim) with
    trees (batch, kv_heads, nodes, head_dim), or both with a leading layers
    dimension: all layers are then written in one launch.  Trees that overlap
    the caches (drafts kept among their rows) are copied first.  Rows are copied as
    data, no gradient goes through the cache.  Rows that the cache has no room
    for are left out and the returned length stops at ``seq_kv``; ``path_lens``
    outside 0..nodes and ``kv_lens`` outside 0..seq_kv are clamped; in either case
    :func:`tklab.kernels.flash_attention.check_device_status` raises.
    """
    args = (k_cache, v_cache, k_tree, v_tree, path, path_lens, kv_lens)
    new_lens = binding.commit_draft(*args)
    if new_lens is None:
        new_lens = binding.commit_draft(*_prepare_commit(*args))
        if new_lens is None:
            raise ValueError("commit: unsupported arguments")
    _after_launch(k_cache.device)
    return new_lens
