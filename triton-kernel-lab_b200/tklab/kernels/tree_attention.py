"""Attention of a tree of drafted tokens over a key/value cache (B200).

The verification pass of speculative decoding: every drafted token of a
sequence is a query at once.  The tokens form a tree (a chain when
``parents`` is None): node 0 is the last token the sequence knows, node ``t``
continues node ``parents[t] < t``.  Query heads share KV heads as in
:func:`tklab.kernels.gqa_decode.gqa_decode`; node ``t`` attends the sequence's
first ``kv_lens[b]`` cache rows, its ancestors and itself.  The tree's own keys
and values are passed beside the cache and stay out of it until
:func:`tklab.kernels.speculative.commit_draft` writes the accepted ones.
"""

from __future__ import annotations

import math

import torch

from tklab._tensors import binding, contiguous, dense, distinct, require_cache
from tklab.kernels.flash_attention import _NATIVE_DTYPE, _after_launch

MAX_TREE_NODES = 256


def check_parents(parents: torch.Tensor | None, batch: int, nodes: int, device: torch.device) -> None:
    """Check optional parents."""
    if parents is None:
        return
    if parents.dtype != torch.int32 or parents.device != device or parents.shape not in ((batch, nodes), (nodes,)):
        raise ValueError("parents must be an int32 tensor of shape (batch, nodes) or (nodes,) on the same device")


def check_lens(lens: torch.Tensor | None, name: str, batch: int, device: torch.device) -> None:
    """Check an optional (batch,) int32 tensor."""
    if lens is not None and (lens.shape != (batch,) or lens.dtype != torch.int32 or lens.device != device):
        raise ValueError(f"{name} must be an int32 tensor of shape (batch,) on the same device")


def _prepare(q, k_cache, v_cache, k_tree, v_tree, kv_lens, parents, tree_sizes, scale) -> tuple:
    """Check the contract; return the arguments with whatever the kernel cannot read in place copied."""
    if q.ndim != 4 or k_cache.ndim != 4 or k_tree.ndim != 4:
        raise ValueError("q, the caches and the tree's keys and values must be 4-dimensional")
    batch, q_heads, nodes, head_dim = q.shape
    kv_heads, seq_kv = k_cache.shape[1], k_cache.shape[2]
    if k_cache.shape != v_cache.shape or k_cache.shape[0] != batch or k_cache.shape[3] != head_dim:
        raise ValueError("K and V caches must be identical (batch, kv_heads, seq_kv, head_dim) tensors")
    if k_tree.shape != v_tree.shape or k_tree.shape != (batch, kv_heads, nodes, head_dim):
        raise ValueError("the tree's keys and values must be (batch, kv_heads, nodes, head_dim) tensors")
    if 0 in q.shape or 0 in k_cache.shape:
        raise ValueError("tree attention does not support empty dimensions")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if nodes > MAX_TREE_NODES:
        raise ValueError(f"tree attention supports up to {MAX_TREE_NODES} nodes")
    if head_dim % 8 or head_dim > 128:
        raise ValueError("tree attention requires head_dim to be a multiple of 8 up to 128")
    dtype = q.dtype
    if dtype not in _NATIVE_DTYPE or not dtype == k_cache.dtype == v_cache.dtype == k_tree.dtype == v_tree.dtype:
        raise ValueError("q, keys and values must share one dtype: float16 or bfloat16")
    device = q.device
    if not device == k_cache.device == v_cache.device == k_tree.device == v_tree.device:
        raise ValueError("q, keys and values must be on the same device")
    if device.type != "cuda":
        raise ValueError("tree attention requires CUDA tensors")
    if scale is not None and not (math.isfinite(scale) and scale > 0.0):
        raise ValueError("scale must be a positive finite number")
    if kv_lens is None:
        raise ValueError("kv_lens is required")
    check_lens(kv_lens, "kv_lens", batch, device)
    check_lens(tree_sizes, "tree_sizes", batch, device)
    check_parents(parents, batch, nodes, device)
    require_cache(k_cache, "the K cache")
    require_cache(v_cache, "the V cache")
    return (
        dense(q.contiguous()), k_cache, v_cache, distinct(k_tree), distinct(v_tree), kv_lens.contiguous(), contiguous(parents),
        contiguous(tree_sizes), scale,
    )


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    kv_lens: torch.Tensor,
    parents: torch.Tensor | None = None,
    *,
    tree_sizes: torch.Tensor | None = None,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``softmax(scale q . K^T) V`` of every node over the cache, its ancestors and itself.

    Args:
        q: (batch, q_heads, nodes, head_dim), 1 to 256 nodes, head_dim a
            multiple of 8 up to 128, float16 or bfloat16.
        k_cache, v_cache: (batch, kv_heads, seq_kv, head_dim), any strides with
            contiguous 16-byte aligned rows; rows past ``kv_lens`` may hold anything.
        k_tree, v_tree: (batch, kv_heads, nodes, head_dim); for a node, the rows that it does not attend may hold anything.
        kv_lens: (batch,) int32, valid cache rows.
        parents: (batch, nodes) or (nodes,) int32, ``parents[t] < t`` (anything
            else makes ``t`` a root); None: a chain.
        tree_sizes: (batch,) int32, nodes in use; the rest get 0 and an lse of -inf.
        scale: default ``1 / sqrt(head_dim)``.

    It serves inference: there is no derivative, and a backward pass that
    reaches it raises.

    Returns ``o`` shaped like ``q`` (and the base-2 log-sum-exp, scale
    included, (batch, q_heads, nodes) fp32 when ``return_lse``).
    """
    args = (q, k_cache, v_cache, k_tree, v_tree, kv_lens, parents, tree_sizes, scale)
    out = binding.tree_attention(*args, return_lse)
    if out is None:
        out = binding.tree_attention(*_prepare(*args), return_lse)
        if out is None:
            raise ValueError("tree attention: unsupported arguments")
    _after_launch(q.device)
    return out
