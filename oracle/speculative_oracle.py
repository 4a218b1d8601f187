"""64-bit CPU references of the speculative-decoding operators, straight from
their definitions, one row at a time (test infrastructure only)."""

from __future__ import annotations

import math

import torch


def rotary_reference(x, cos, sin, *, positions=None, layout="half", transpose=False):
    """Rotate (batch, heads, seq, dim) ``x`` in 64 bits; rows at positions outside the tables are kept."""
    half = cos.shape[1]
    y = x.double().clone()
    for b in range(x.shape[0]):
        for s in range(x.shape[2]):
            p = s if positions is None else int(positions[b, s])
            if not 0 <= p < cos.shape[0]:
                continue
            c, t = cos[p].double(), sin[p].double() * (-1.0 if transpose else 1.0)
            row = x[b, :, s].double()
            if layout == "half":
                first, second = row[:, :half], row[:, half : 2 * half]
                y[b, :, s, :half], y[b, :, s, half : 2 * half] = first * c - second * t, second * c + first * t
            else:
                first, second = row[:, 0 : 2 * half : 2], row[:, 1 : 2 * half : 2]
                y[b, :, s, 0 : 2 * half : 2], y[b, :, s, 1 : 2 * half : 2] = first * c - second * t, second * c + first * t
    return y


def lineage(parents, node):
    """``node`` and its ancestors (``parents`` None: a chain)."""
    out = []
    while node >= 0:
        out.append(node)
        up = node - 1 if parents is None else int(parents[node])
        node = up if up < node else -1
    return out


def tree_attention_reference(q, k_cache, v_cache, k_tree, v_tree, kv_lens, parents=None, *, tree_sizes=None, scale=None):
    """(o, base-2 lse, spread) in 64 bits; ``spread`` is the same average of ``|v|``, the scale of o's rounding errors."""
    batch, q_heads, nodes, dim = q.shape
    kv_heads, capacity = k_cache.shape[1], k_cache.shape[2]
    group = q_heads // kv_heads
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64)
    spread = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    for b in range(batch):
        n = min(max(int(kv_lens[b]), 0), capacity)
        size = nodes if tree_sizes is None else min(max(int(tree_sizes[b]), 0), nodes)
        tree = None if parents is None else (parents if parents.ndim == 1 else parents[b])
        for t in range(size):
            own = sorted(lineage(tree, t))
            for h in range(kv_heads):
                keys = torch.cat((k_cache[b, h, :n], k_tree[b, h, own])).double()
                values = torch.cat((v_cache[b, h, :n], v_tree[b, h, own])).double()
                heads = slice(h * group, (h + 1) * group)
                scores = scale * q[b, heads, t].double() @ keys.T
                weights = torch.softmax(scores, -1)
                o[b, heads, t] = weights @ values
                spread[b, heads, t] = weights @ values.abs()
                lse[b, heads, t] = torch.logsumexp(scores, -1) / math.log(2.0)
    return o, lse, spread


def verify_reference(target, tokens, uniforms, noise, *, parents=None, draft=None, tree_sizes=None):
    """(path, path_lens, next) of :func:`tklab.kernels.speculative.verify_draft` in 64 bits."""
    batch, nodes, vocab = target.shape
    path = torch.full((batch, nodes), -1, dtype=torch.int32)
    lens = torch.zeros(batch, dtype=torch.int32)
    nexts = torch.full((batch,), -1, dtype=tokens.dtype)
    for b in range(batch):
        size = nodes if tree_sizes is None else min(max(int(tree_sizes[b]), 0), nodes)
        if size == 0:
            continue
        tree = None if parents is None else (parents if parents.ndim == 1 else parents[b])
        walk = [0]
        while True:
            node = walk[-1]
            p = torch.nan_to_num(target[b, node].double(), nan=0.0)
            weights, tried, accepted = p.clone(), set(), None
            children = [c for c in range(node + 1, size) if (c - 1 if tree is None else int(tree[c])) == node]
            if children and draft is not None:
                weights = torch.nan_to_num(p - draft[b, node].double(), nan=0.0).clamp_min(0.0)
            for c in children:
                x, u = int(tokens[b, c]), float(uniforms[b, c])
                inside = 0 <= x < vocab
                px = float(p[x]) if inside else 0.0
                if draft is not None:
                    passed = inside and px > 0.0 and u * float(draft[b, node, x]) < px
                else:
                    mass = sum(float(p[t]) for t in tried if 0 <= t < vocab)
                    passed = px > 0.0 and x not in tried and u * max(1.0 - mass, 0.0) < px
                    tried.add(x)
                    if inside:
                        weights[x] = 0.0
                if passed:
                    accepted = c
                    break
            if accepted is None:
                break
            walk.append(accepted)
        if not bool((weights > 0.0).any()):
            weights = p
        path[b, : len(walk)] = torch.tensor(walk, dtype=torch.int32)
        lens[b] = len(walk)
        nexts[b] = int((weights.clamp_min(0.0) / noise[b].double()).argmax())
    return path, lens, nexts


def commit_reference(k_cache, v_cache, k_tree, v_tree, path, path_lens, kv_lens):
    """New (k_cache, v_cache, kv_lens); tensors with a leading layers dimension."""
    k_cache, v_cache, lens = k_cache.clone(), v_cache.clone(), kv_lens.clone()
    capacity = k_cache.shape[3]
    for b in range(k_cache.shape[1]):
        start = min(max(int(kv_lens[b]), 0), capacity)
        n = min(int(path_lens[b]), capacity - start)
        for i in range(n):
            k_cache[:, b, :, start + i] = k_tree[:, b, :, int(path[b, i])]
            v_cache[:, b, :, start + i] = v_tree[:, b, :, int(path[b, i])]
        lens[b] = start + n
    return k_cache, v_cache, lens
