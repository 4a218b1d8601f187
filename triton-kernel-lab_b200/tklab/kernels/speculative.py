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

from tklab import _native
from tklab.kernels._plans import Plans, _after_launch, _stream, at_device, dense, meta, row_strides, stride_array
from tklab.kernels.flash_attention import _NATIVE_DTYPE
from tklab.kernels.tree_attention import MAX_TREE_NODES, check_lens, check_parents, in_place

_PROB_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_TOKEN_TYPES = (torch.int32, torch.int64)
_VERIFY_PLANS, _COMMIT_PLANS = Plans(), Plans()


class Verification(NamedTuple):
    """What :func:`verify_draft` found for each sequence of the batch."""

    path: torch.Tensor  # (batch, nodes) int32: the accepted nodes from node 0 on, then -1
    path_lens: torch.Tensor  # (batch,) int32: how many (node 0 counts)
    next_tokens: torch.Tensor  # (batch,), the tokens' dtype


def _verify_plan(target_probs, tokens, uniforms, noise, parents, draft_probs, tree_sizes) -> tuple:
    """Check the contract; return what a call with this metadata passes to the library.

    The first entry says whether every tensor can be read in place.
    """
    if target_probs.ndim != 3 or 0 in target_probs.shape:
        raise ValueError("target_probs must be a non-empty (batch, nodes, vocab) tensor")
    batch, nodes, vocab = target_probs.shape
    if nodes > MAX_TREE_NODES:
        raise ValueError(f"verification supports up to {MAX_TREE_NODES} nodes")
    if target_probs.dtype not in _PROB_TYPE:
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
    parent_stride = check_parents(parents, batch, nodes, device)
    check_lens(tree_sizes, "tree_sizes", batch, device)
    drafted = draft_probs is not None and nodes > 1
    ready = (
        (target_probs.stride(2) == 1 or vocab == 1)
        and (not drafted or draft_probs.stride(2) == 1 or vocab == 1)
        and all(x is None or x.is_contiguous() for x in (tokens, uniforms, noise, parents, tree_sizes))
    )
    return (
        ready, target_probs.get_device(), stride_array(*target_probs.stride()[:2]), drafted,
        stride_array(*draft_probs.stride()[:2]) if drafted else None, int(tokens.dtype == torch.int64), parent_stride,
        batch, nodes, vocab, _PROB_TYPE[target_probs.dtype],
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
    key = (
        target_probs.shape, target_probs.stride(), target_probs.dtype, target_probs.get_device(), tokens.shape,
        tokens.stride(), tokens.dtype, tokens.get_device(), uniforms.shape, uniforms.stride(), uniforms.dtype,
        uniforms.get_device(), noise.shape, noise.stride(), noise.dtype, noise.get_device(), meta(parents),
        meta(draft_probs), meta(tree_sizes),
    )
    plan = _VERIFY_PLANS.get(key) or _VERIFY_PLANS.keep(
        key, _verify_plan(target_probs, tokens, uniforms, noise, parents, draft_probs, tree_sizes)
    )
    (ready, device, target_strides, drafted, draft_strides, wide, parent_stride, batch, nodes, vocab, prob_type) = plan
    if not ready:
        return verify_draft(
            target_probs.contiguous(), tokens.contiguous(), uniforms.contiguous(), noise.contiguous(),
            parents=None if parents is None else parents.contiguous(),
            draft_probs=None if draft_probs is None else draft_probs.contiguous(),
            tree_sizes=None if tree_sizes is None else tree_sizes.contiguous(),
        )
    path = torch.empty_like(uniforms, dtype=torch.int32)
    path_lens = uniforms.new_empty((batch,), dtype=torch.int32)
    next_tokens = tokens.new_empty((batch,))
    with at_device(device):
        status = _native.load().tk_verify_draft(
            target_probs.data_ptr(), target_strides, draft_probs.data_ptr() if drafted else 0, draft_strides,
            tokens.data_ptr(), wide, 0 if parents is None else parents.data_ptr(), parent_stride,
            0 if tree_sizes is None else tree_sizes.data_ptr(), uniforms.data_ptr(), noise.data_ptr(),
            path.data_ptr(), path_lens.data_ptr(), next_tokens.data_ptr(), batch, nodes, vocab, prob_type,
            _stream(target_probs),
        )
    _native.check(status, "tk_verify_draft")
    _after_launch(target_probs.device)
    return Verification(path, path_lens, next_tokens)


def _commit_plan(k_cache, v_cache, k_tree, v_tree, path, path_lens, kv_lens) -> tuple:
    """Check the contract; return what a call with this metadata passes to the library.

    The first entry says whether every tensor can be read in place.
    """
    if not k_cache.ndim == v_cache.ndim == k_tree.ndim == v_tree.ndim or k_cache.ndim not in (4, 5) or (
        k_cache.shape != v_cache.shape or k_tree.shape != v_tree.shape
    ):
        raise ValueError(
            "K and V caches, and the tree's keys and values, must have identical shapes: ([layers,] batch, heads, rows, dim)"
        )
    if k_cache.ndim == 4:
        k_cache, v_cache, k_tree, v_tree = k_cache[None], v_cache[None], k_tree[None], v_tree[None]
    layers, batch, kv_heads, seq_kv, head_dim = k_cache.shape
    nodes = k_tree.shape[3]
    if k_tree.shape != (layers, batch, kv_heads, nodes, head_dim):
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
    caches = in_place(k_cache, "the K cache") + in_place(v_cache, "the V cache")
    trees = [row_strides(k_tree), row_strides(v_tree)]
    ready = None not in trees and all(x.is_contiguous() for x in (path, path_lens, kv_lens))
    return (
        ready, k_cache.get_device(), stride_array(*caches, *trees[0], *trees[1]) if ready else None,
        layers, batch, kv_heads, nodes, seq_kv, head_dim,
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
    dimension: all layers are then written in one launch.  Rows that the cache
    has no room for are left out, the returned length stops at ``seq_kv`` and
    :func:`tklab.kernels.flash_attention.check_device_status` raises.
    """
    key = (
        k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.get_device(), v_cache.shape, v_cache.stride(),
        v_cache.dtype, v_cache.get_device(), k_tree.shape, k_tree.stride(), k_tree.dtype, k_tree.get_device(),
        v_tree.shape, v_tree.stride(), v_tree.dtype, v_tree.get_device(), path.shape, path.stride(), path.dtype,
        path.get_device(), path_lens.shape, path_lens.stride(), path_lens.dtype, path_lens.get_device(), kv_lens.shape,
        kv_lens.stride(), kv_lens.dtype, kv_lens.get_device(),
    )
    plan = _COMMIT_PLANS.get(key) or _COMMIT_PLANS.keep(
        key, _commit_plan(k_cache, v_cache, k_tree, v_tree, path, path_lens, kv_lens)
    )
    ready, device, strides, layers, batch, kv_heads, nodes, seq_kv, head_dim = plan
    k_ptr, v_ptr, kt_ptr, vt_ptr = k_cache.data_ptr(), v_cache.data_ptr(), k_tree.data_ptr(), v_tree.data_ptr()
    if (k_ptr | v_ptr) & 15:
        raise ValueError("the caches need contiguous, 16-byte aligned rows at distinct strides that are multiples of 8")
    if not ready or (kt_ptr | vt_ptr) & 15:
        return commit_draft(
            k_cache, v_cache, dense(k_tree), dense(v_tree), path.contiguous(), path_lens.contiguous(), kv_lens.contiguous()
        )
    new_lens = torch.empty_like(kv_lens)
    with at_device(device):
        status = _native.load().tk_commit_draft(
            k_ptr, v_ptr, kt_ptr, vt_ptr, strides, path.data_ptr(), path_lens.data_ptr(), kv_lens.data_ptr(),
            new_lens.data_ptr(), layers, batch, kv_heads, nodes, seq_kv, head_dim, _stream(k_cache),
        )
    _native.check(status, "tk_commit_draft")
    _after_launch(k_cache.device)
    return new_lens
