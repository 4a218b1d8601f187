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

import ctypes
import functools
import math

import torch

from tklab import _native
from tklab.kernels.flash_attention import _NATIVE_DTYPE, _after_launch, _on_device, _stream

MAX_TREE_NODES = 256
TREE_HEAD_DIMS = tuple(range(8, 129, 8))


@functools.lru_cache(maxsize=1024)
def _stride_array(*strides: int) -> ctypes.Array:
    """Strides as the C array that the library reads (never written)."""
    return (ctypes.c_int64 * len(strides))(*strides)


def _row_strides(x: torch.Tensor) -> tuple[int, ...] | None:
    """Strides of every dimension but the last (0 for dimensions of size 1), or None if rows cannot be read in place."""
    *outer, last = x.stride()
    if (last != 1 and x.shape[-1] > 1) or x.data_ptr() & 15:
        return None
    strides = tuple(0 if n == 1 else s for n, s in zip(x.shape, outer))
    return None if any(s % 8 or (s == 0 and n > 1) for s, n in zip(strides, x.shape)) else strides


def _in_place(x: torch.Tensor, name: str) -> tuple[int, ...]:
    strides = _row_strides(x)
    if strides is None:
        raise ValueError(f"{name} needs contiguous, 16-byte aligned rows at strides that are multiples of 8")
    return strides


def _or_copy(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """``x`` and its strides, copied first if its rows cannot be read in place."""
    strides = _row_strides(x)
    if strides is None:
        x = x.clone(memory_format=torch.contiguous_format)
        strides = _row_strides(x)
    return x, strides


def _check_parents(parents: torch.Tensor | None, batch: int, nodes: int, device: torch.device) -> tuple[torch.Tensor | None, int]:
    """The parents (int32, (batch, nodes) or (nodes,)) and their batch stride (0: one tree for all)."""
    if parents is None:
        return None, 0
    if parents.dtype != torch.int32 or parents.device != device or parents.shape not in ((batch, nodes), (nodes,)):
        raise ValueError("parents must be an int32 tensor of shape (batch, nodes) or (nodes,) on the same device")
    return parents.contiguous(), nodes if parents.ndim == 2 else 0


def _check_lens(lens: torch.Tensor | None, name: str, batch: int, device: torch.device) -> torch.Tensor | None:
    if lens is None:
        return None
    if lens.shape != (batch,) or lens.dtype != torch.int32 or lens.device != device:
        raise ValueError(f"{name} must be an int32 tensor of shape (batch,) on the same device")
    return lens.contiguous()


@functools.lru_cache(maxsize=512)
def _workspace_bytes(lib, device_index, batch, q_heads, kv_heads, nodes, seq_kv, head_dim) -> int:
    """Scratch bytes for this shape on this device."""
    return int(lib.tk_tree_attn_workspace_bytes(batch, q_heads, kv_heads, nodes, seq_kv, head_dim))


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
        k_tree, v_tree: (batch, kv_heads, nodes, head_dim).
        kv_lens: (batch,) int32, valid cache rows.
        parents: (batch, nodes) or (nodes,) int32, ``parents[t] < t`` (anything
            else makes ``t`` a root); None: a chain.
        tree_sizes: (batch,) int32, nodes in use; the rest get 0 and an lse of -inf.
        scale: default ``1 / sqrt(head_dim)``.

    Returns ``o`` shaped like ``q`` (and the base-2 log-sum-exp, scale
    included, (batch, q_heads, nodes) fp32 when ``return_lse``).
    """
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
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    elif not (math.isfinite(scale) and scale > 0.0):
        raise ValueError("scale must be a positive finite number")
    kv_lens = _check_lens(kv_lens, "kv_lens", batch, device)
    if kv_lens is None:
        raise ValueError("kv_lens is required")
    tree_sizes = _check_lens(tree_sizes, "tree_sizes", batch, device)
    parents, parent_stride = _check_parents(parents, batch, nodes, device)
    strides = _in_place(k_cache, "the K cache") + _in_place(v_cache, "the V cache")
    k_tree, k_strides = _or_copy(k_tree)
    v_tree, v_strides = _or_copy(v_tree)
    q = q.contiguous()
    if q.data_ptr() & 15:
        q = q.clone()
    lib = _native.load()
    out = torch.empty((batch, q_heads, nodes, head_dim), dtype=dtype, device=device)
    lse = torch.empty((batch, q_heads, nodes), dtype=torch.float32, device=device) if return_lse else None
    with _on_device(device):
        ws_bytes = _workspace_bytes(lib, device.index, batch, q_heads, kv_heads, nodes, seq_kv, head_dim)
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        status = lib.tk_tree_attn(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_tree.data_ptr(), v_tree.data_ptr(),
            _stride_array(*strides, *k_strides, *v_strides), kv_lens.data_ptr(),
            None if parents is None else parents.data_ptr(), parent_stride,
            None if tree_sizes is None else tree_sizes.data_ptr(), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if workspace is None else workspace.data_ptr(), ws_bytes,
            batch, q_heads, kv_heads, nodes, seq_kv, head_dim, _NATIVE_DTYPE[dtype], scale, _stream(q),
        )
    _native.check(status, "tk_tree_attn")
    _after_launch(device)
    return (out, lse) if return_lse else out
