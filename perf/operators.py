"""Measured cases of the speculative-decoding operators.

Four operators, each with a plain form (elementary torch operations, 32 bits,
rounded once) and the framework's own call:

rotary          rotary positions on queries and keys, forward (+ backward)
tree_attention  attention of a tree of drafted tokens over a key/value cache
verify          acceptance of drafted tokens and the draw of the next token
commit          the accepted tokens' keys and values written into the cache

``prepare`` makes the same state for both forms; ``run`` is one pass.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_PACKAGE = str(Path(__file__).resolve().parents[1] / "triton-kernel-lab_b200")


def listed():
    """The measured cases, smallest and largest calls of each operator among them."""
    return [
        # Training at a long sequence: whole heads, projection output order (batch, seq, heads, dim), both directions.
        {"name": "rotary_train_16k", "op": "rotary", "batch": 1, "q_heads": 32, "kv_heads": 8, "seq": 16384, "dim": 128,
         "rotary_dim": 128, "layout": "half", "dtype": "bf16", "train": True, "order": "bshd", "positions": False},
        # Training at an odd length with a quarter of the head rotated in adjacent pairs, both directions.
        {"name": "rotary_train_part", "op": "rotary", "batch": 3, "q_heads": 16, "kv_heads": 16, "seq": 2047, "dim": 96,
         "rotary_dim": 24, "layout": "interleaved", "dtype": "f16", "train": True, "order": "bhsd", "positions": False},
        # Serving: the drafted tokens of every sequence of a batch, each at its own depth's position.
        {"name": "rotary_draft", "op": "rotary", "batch": 32, "q_heads": 32, "kv_heads": 8, "seq": 24, "dim": 128,
         "rotary_dim": 128, "layout": "half", "dtype": "bf16", "train": False, "order": "bshd", "positions": True},
        # The smallest serving call: one sequence, a short cache, a handful of drafted tokens; latency counts.
        {"name": "tree_one_sequence", "op": "tree", "batch": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "tree": 8,
         "cache": 1024, "len_min": 700, "len_max": 1000, "dtype": "bf16", "chain": False},
        # A batch with ragged lengths and a wide tree: rows fill the tensor cores, about balanced with the cache's bytes.
        {"name": "tree_batch_wide", "op": "tree", "batch": 32, "q_heads": 32, "kv_heads": 8, "dim": 128, "tree": 64,
         "cache": 8192, "len_min": 4096, "len_max": 8192, "dtype": "bf16", "chain": False},
        # Two long conversations: the cache is read once, split over the whole device.
        {"name": "tree_long_cache", "op": "tree", "batch": 2, "q_heads": 32, "kv_heads": 4, "dim": 128, "tree": 13,
         "cache": 131072, "len_min": 100000, "len_max": 131000, "dtype": "f16", "chain": False},
        # Heads without sharing, 64 wide, a short drafted chain, lengths from nothing to a full cache.
        {"name": "tree_chain_64", "op": "tree", "batch": 24, "q_heads": 16, "kv_heads": 16, "dim": 64, "tree": 5,
         "cache": 4096, "len_min": 0, "len_max": 4096, "dtype": "bf16", "chain": True},
        # One sequence's drafted chain against its target: the smallest call.
        {"name": "verify_one_chain", "op": "verify", "batch": 1, "tree": 6, "vocab": 32000, "dtype": "f32", "chain": True, "draft": True},
        # A serving batch of chains with the draft's own probabilities, odd vocabulary.
        {"name": "verify_batch_chain", "op": "verify", "batch": 128, "tree": 5, "vocab": 50257, "dtype": "f32", "chain": True, "draft": True},
        # A serving batch of trees over a large vocabulary, 16-bit probabilities.
        {"name": "verify_batch_tree", "op": "verify", "batch": 32, "tree": 64, "vocab": 128000, "dtype": "bf16", "chain": False, "draft": False},
        # One sequence's accepted tokens into one layer's cache: the smallest call.
        {"name": "commit_one_layer", "op": "commit", "layers": 1, "batch": 1, "kv_heads": 8, "dim": 128, "tree": 8, "cache": 2048, "dtype": "bf16"},
        # Every layer of a serving batch at once, long accepted paths.
        {"name": "commit_all_layers", "op": "commit", "layers": 32, "batch": 32, "kv_heads": 8, "dim": 128, "tree": 32, "cache": 256, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["rotary", "rotary", "tree", "tree", "tree", "verify", "verify", "commit"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rotary":
        train = rng.random() < 0.5
        dim = rng.choice([64, 80, 96, 128, 128])
        rotary_dim = rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2])
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        q_heads = kv_heads * rng.choice([1, 2, 3, 4])
        tokens = _log(rng, 16, 13000 * 40 * 128 // ((q_heads + kv_heads) * dim * (1 if train else 4)))
        seq = min(tokens, _log(rng, 1, 16384))
        return {"op": op, "batch": max(1, min(256, tokens // seq)), "q_heads": q_heads, "kv_heads": kv_heads, "seq": seq, "dim": dim,
                "rotary_dim": rotary_dim, "layout": rng.choice(["half", "interleaved"]), "dtype": dtype, "train": train,
                "order": rng.choice(["bshd", "bhsd"]), "positions": rng.random() < 0.5}
    if op == "tree":
        dim = rng.choice([64, 96, 128, 128])
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        tree = _log(rng, 1, 128)
        cache = _log(rng, 64, 131072)
        most = min(32 * 8 * 8192 * 128 // (kv_heads * cache * dim), 32 * 32 * 64 * 8192 // (kv_heads * group * tree * cache))
        if most < 1:
            kv_heads, group, most = 1, 4, max(1, 32 * 32 * 64 * 8192 // (4 * tree * cache))
        len_max = rng.randint(cache // 2, cache)
        return {"op": op, "batch": _log(rng, 1, max(1, min(64, most))), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "tree": tree, "cache": cache, "len_min": rng.choice([0, len_max // 2]), "len_max": len_max, "dtype": dtype,
                "chain": rng.random() < 0.3}
    if op == "verify":
        chain = rng.random() < 0.5
        draft = chain and rng.random() < 0.7
        vocab = _log(rng, 1000, 200000)
        tree = rng.randint(1, 12) if chain else _log(rng, 2, 64)
        most = 32 * 64 * 128000 // (vocab * tree * (4 if draft else 2))
        return {"op": op, "batch": _log(rng, 1, max(1, min(128, most))), "tree": tree, "vocab": vocab,
                "dtype": rng.choice(["f32", "bf16", "f16"]), "chain": chain, "draft": draft}
    cache = _log(rng, 64, 2048)
    batch, kv_heads, dim = _log(rng, 1, 32), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 128])
    most = 32 * 32 * 8 * 256 * 128 // (batch * kv_heads * cache * dim)
    return {"op": op, "layers": _log(rng, 1, max(1, min(48, most))), "batch": batch, "kv_heads": kv_heads, "dim": dim,
            "tree": _log(rng, 1, min(64, cache)), "cache": cache, "dtype": dtype}


# --------------------------------------------------------------------------
# What a program has in hand before the call.
# --------------------------------------------------------------------------
def _randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _parents(gen, batch, tree):
    """Random trees in topological order, leaning towards depth: parent[i] < i, parent[0] = -1."""
    index = torch.arange(tree, device="cuda")
    u = torch.rand(batch, tree, generator=gen, device="cuda").sqrt()
    parents = torch.minimum((u * index).floor(), (index - 1).clamp_min(0)).to(torch.int32)
    parents[:, 0] = -1
    return parents


def prepare(case, seed):
    """Inputs of one pass, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "rotary":
        batch, seq, dim = case["batch"], case["seq"], case["dim"]
        limit = max(seq, 4096)
        rates = 10000.0 ** (-torch.arange(0, case["rotary_dim"], 2, device="cuda", dtype=torch.float64) / case["rotary_dim"])
        angles = torch.arange(limit, device="cuda", dtype=torch.float64)[:, None] * rates
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        state["pos"] = None
        if case["positions"]:
            start = torch.randint(0, limit - seq + 1, (batch, 1), generator=gen, device="cuda")
            depth = torch.randint(0, seq, (batch, seq), generator=gen, device="cuda").sort(dim=1).values
            state["pos"] = (start + depth).to(torch.int32)
        for name, heads in (("q", case["q_heads"]), ("k", case["kv_heads"])):
            if case["order"] == "bshd":
                state[name] = _randn(gen, dtype, batch, seq, heads, dim).transpose(1, 2)
            else:
                state[name] = _randn(gen, dtype, batch, heads, seq, dim)
            if case["train"]:
                state[name].requires_grad_(True)
                state["d" + name] = _randn(gen, dtype, batch, heads, seq, dim)
    elif case["op"] == "tree":
        batch, heads, dim, tree = case["batch"], case["kv_heads"], case["dim"], case["tree"]
        state["q"] = _randn(gen, dtype, batch, case["q_heads"], tree, dim)
        for name in ("k", "v"):
            state[name + "_cache"] = _randn(gen, dtype, batch, heads, case["cache"], dim)
            state[name + "_tree"] = _randn(gen, dtype, batch, heads, tree, dim)
        state["lens"] = torch.randint(case["len_min"], case["len_max"] + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
        state["parents"] = None if case["chain"] else _parents(gen, batch, tree)
    elif case["op"] == "verify":
        batch, tree, vocab = case["batch"], case["tree"], case["vocab"]
        logits = 4.0 * torch.randn(batch, tree, vocab, generator=gen, device="cuda")
        state["target"] = logits.softmax(-1).to(dtype)
        source, state["draft_probs"] = state["target"], None
        if case["draft"]:
            near = logits[:, : tree - 1] + 0.7 * torch.randn(batch, tree - 1, vocab, generator=gen, device="cuda")
            source = state["draft_probs"] = near.softmax(-1).to(dtype)
        state["parents"] = None if case["chain"] else _parents(gen, batch, tree)
        # Each drafted token is a draw from the distribution at its parent.
        at = torch.arange(-1, tree - 1, device="cuda").expand(batch, tree) if case["chain"] else state["parents"]
        race = torch.empty(batch, tree, vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-9)
        tokens = torch.randint(0, vocab, (batch, tree), generator=gen, device="cuda")
        if tree > 1:
            rows = at[:, 1:].long()[..., None].expand(-1, -1, vocab)
            tokens[:, 1:] = (source.gather(1, rows).float() / race[:, 1:]).argmax(-1)
        state["tokens"] = tokens
        state["uniforms"] = torch.rand(batch, tree, generator=gen, device="cuda")
        state["noise"] = torch.empty(batch, vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-9)
    else:
        layers, batch, heads, dim, tree, cache = (case[n] for n in ("layers", "batch", "kv_heads", "dim", "tree", "cache"))
        for name in ("k", "v"):
            state[name + "_cache"] = _randn(gen, dtype, layers, batch, heads, cache, dim)
            state[name + "_tree"] = _randn(gen, dtype, layers, batch, heads, tree, dim)
        # A path of 1..tree increasing nodes from the root, about half of them on average.
        length = torch.randint(1, tree + 1, (batch, 1), generator=gen, device="cuda")
        order = torch.rand(batch, tree, generator=gen, device="cuda")
        order[:, 0] = -1.0
        index = torch.arange(tree, device="cuda")
        kept = order.argsort(1).argsort(1) < length
        path = torch.where(kept, index, tree).sort(1).values
        state["path"] = torch.where(path < tree, path, -1).to(torch.int32)
        state["path_lens"] = length[:, 0].to(torch.int32)
        state["lens"] = torch.randint(0, cache - tree + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    return state


# --------------------------------------------------------------------------
# The plain forms.
# --------------------------------------------------------------------------
def _split_pairs(x, layout):
    return x.chunk(2, dim=-1) if layout == "half" else (x[..., 0::2], x[..., 1::2])


def _join_pairs(first, second, layout):
    return torch.cat((first, second), -1) if layout == "half" else torch.stack((first, second), -1).flatten(-2)


def _plain_rotate(x, cos, sin, rotary_dim, layout):
    first, second = _split_pairs(x[..., :rotary_dim].float(), layout)
    turned = _join_pairs(first * cos - second * sin, second * cos + first * sin, layout)
    return torch.cat((turned, x[..., rotary_dim:].float()), -1).to(x.dtype)


def _plain_rotary(s):
    if s["pos"] is None:
        cos, sin = s["cos"][: s["seq"]], s["sin"][: s["seq"]]
    else:
        cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    args = (s["rotary_dim"], s["layout"])
    with torch.no_grad():
        out = [_plain_rotate(s["q"], cos, sin, *args), _plain_rotate(s["k"], cos, sin, *args)]
        if s["train"]:
            out += [_plain_rotate(s["dq"], cos, -sin, *args), _plain_rotate(s["dk"], cos, -sin, *args)]
    return out


def _lineage(parents):
    """(batch, T, T) truth values: node j is node i or one of its ancestors."""
    tree = parents.shape[1]
    index = torch.arange(tree, device=parents.device)
    edge = (parents[:, :, None] == index).float()  # [i, j]: j is i's parent
    eye = torch.eye(tree, device=parents.device)
    # (I - E)^-1 = I + E + E^2 + ... for the strictly lower triangular E.
    return torch.linalg.solve_triangular(eye - edge, eye.expand_as(edge), upper=False, unitriangular=True) > 0.5


def _chain(batch, tree):
    return torch.arange(-1, tree - 1, device="cuda", dtype=torch.int32).expand(batch, tree)


def _plain_tree(s):
    batch, heads, tree, dim, cache = s["batch"], s["kv_heads"], s["tree"], s["dim"], s["cache"]
    parents = _chain(batch, tree) if s["parents"] is None else s["parents"]
    rows = s["q"].float().view(batch, heads, -1, dim) * (1.0 / math.sqrt(dim))
    held = torch.arange(cache, device="cuda") < s["lens"][:, None]
    on_cache = (rows @ s["k_cache"].float().transpose(-1, -2)).masked_fill_(~held[:, None, None], -math.inf)
    on_tree = (rows @ s["k_tree"].float().transpose(-1, -2)).view(batch, heads, -1, tree, tree)
    on_tree = on_tree.masked_fill(~_lineage(parents)[:, None, None], -math.inf).view(batch, heads, -1, tree)
    top = torch.maximum(on_cache.amax(-1, keepdim=True), on_tree.amax(-1, keepdim=True))
    on_cache, on_tree = on_cache.sub_(top).exp_(), (on_tree - top).exp()
    total = on_cache.sum(-1, keepdim=True) + on_tree.sum(-1, keepdim=True)
    out = (on_cache @ s["v_cache"].float() + on_tree @ s["v_tree"].float()) / total
    return out.to(s["q"].dtype).view(batch, s["q_heads"], tree, dim)


def _plain_verify(s):
    batch, tree, vocab = s["target"].shape
    parents = (_chain(batch, tree) if s["parents"] is None else s["parents"]).long()
    tokens, index = s["tokens"], torch.arange(tree, device="cuda")
    flat = s["target"].view(batch, tree * vocab)
    up = parents.clamp_min(0)
    prob = flat.gather(1, up * vocab + tokens).float()
    siblings = (parents[:, :, None] == parents[:, None, :]) & (index[:, None] > index)
    if s["draft_probs"] is not None:
        last = max(tree - 2, 0)
        rows = s["draft_probs"].view(batch, -1)
        odds = rows.gather(1, up.clamp_max(last) * vocab + tokens).float() if tree > 1 else torch.ones_like(prob)
        passed = s["uniforms"] * odds < prob
    else:
        again = (siblings & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
        prob = prob.masked_fill(again, 0.0)
        rest = (1.0 - (siblings * prob[:, None, :]).sum(-1)).clamp_min(0.0)
        passed = s["uniforms"] * rest < prob
    passed[:, 0] = True
    chosen = passed & ~(siblings & passed[:, None, :]).any(-1)
    reached = (chosen[:, None, :] | ~_lineage(parents)).all(-1)
    path = torch.where(reached, index, tree).sort(1).values
    last = torch.where(reached, index, 0).amax(1)
    pick = torch.arange(batch, device="cuda")
    row = s["target"][pick, last].float()
    child = parents == last[:, None]
    if s["draft_probs"] is not None and tree > 1:
        drafted = s["draft_probs"][pick, last.clamp_max(tree - 2)].float()
        left = torch.where(child.any(1, keepdim=True), (row - drafted).clamp_min(0.0), row)
    else:
        gone = torch.where(child, tokens, vocab)
        left = torch.cat((row, row[:, :1]), 1).scatter(1, gone, 0.0)[:, :vocab]
    left = torch.where(left.amax(1, keepdim=True) > 0, left, row)
    return [torch.where(path < tree, path, -1).to(torch.int32), reached.sum(1, dtype=torch.int32), (left / s["noise"]).argmax(1)]


def _plain_commit(s):
    layers, batch, heads, tree, dim = s["k_tree"].shape
    index = torch.arange(tree, device="cuda")
    kept = index < s["path_lens"][:, None]
    node = torch.where(kept, s["path"], 0).long()
    slot = (s["lens"][:, None] + torch.where(kept, index, 0)).long()
    pick, head = torch.arange(batch, device="cuda")[:, None, None], torch.arange(heads, device="cuda")[None, :, None]
    # Rows past a path's end repeat its first row, which is written to the same slot.
    s["k_cache"][:, pick, head, slot[:, None]] = s["k_tree"][:, pick, head, node[:, None]]
    s["v_cache"][:, pick, head, slot[:, None]] = s["v_tree"][:, pick, head, node[:, None]]
    return [s["k_cache"], s["v_cache"], s["lens"] + s["path_lens"]]


# --------------------------------------------------------------------------
# One pass.
# --------------------------------------------------------------------------
def _own_rotary(s):
    from tklab.kernels.rotary import rotary

    q, k = rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["pos"], layout=s["layout"])
    if not s["train"]:
        return [q, k]
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]


def _own_tree(s):
    from tklab.kernels.tree_attention import tree_attention

    return tree_attention(s["q"], s["k_cache"], s["v_cache"], s["k_tree"], s["v_tree"], s["lens"], s["parents"])


def _own_verify(s):
    from tklab.kernels.speculative import verify_draft

    return list(verify_draft(s["target"], s["tokens"], s["uniforms"], s["noise"], parents=s["parents"], draft_probs=s["draft_probs"]))


def _own_commit(s):
    from tklab.kernels.speculative import commit_draft

    lens = commit_draft(s["k_cache"], s["v_cache"], s["k_tree"], s["v_tree"], s["path"], s["path_lens"], s["lens"])
    return [s["k_cache"], s["v_cache"], lens]


_PLAIN = {"rotary": _plain_rotary, "tree": _plain_tree, "verify": _plain_verify, "commit": _plain_commit}
_OWN = {"rotary": _own_rotary, "tree": _own_tree, "verify": _own_verify, "commit": _own_commit}


def run(state):
    """One pass through the case's operator and its outputs."""
    if not own:
        return _PLAIN[state["op"]](state)
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    return _OWN[state["op"]](state)


def work(case):
    """Bytes and operations one pass cannot do without (each input read once, each output written once)."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        rows = case["batch"] * (case["q_heads"] + case["kv_heads"]) * case["seq"]
        passes = 2 if case["train"] else 1
        tables = 4 * case["seq"] * case["rotary_dim"] * (case["batch"] if case["positions"] else 1)
        return {"bytes": passes * (2 * size * rows * case["dim"] + tables), "flops": passes * 3 * rows * case["rotary_dim"]}
    if case["op"] == "tree":
        keys = (case["len_min"] + case["len_max"]) / 2 + case["tree"]
        rows = case["batch"] * case["q_heads"] * case["tree"]
        return {"bytes": size * case["dim"] * (2 * case["batch"] * case["kv_heads"] * keys + 2 * rows), "flops": 4 * rows * keys * case["dim"]}
    if case["op"] == "verify":
        per_token = 4 + size * (2 if case["draft"] else 1)
        return {"bytes": case["batch"] * (case["vocab"] * per_token + case["tree"] * (16 + size)), "flops": 2 * case["batch"] * case["vocab"]}
    rows = case["layers"] * case["batch"] * case["kv_heads"] * (case["tree"] + 1) / 2
    return {"bytes": 2 * 2 * size * rows * case["dim"] + 12 * case["batch"], "flops": 0}


# --------------------------------------------------------------------------
# The definitions in 64 bits, one sequence (and one layer) at a time.
# --------------------------------------------------------------------------
def exact(case, seed):
    """What ``run`` returns for these inputs, from the definition in 64 bits."""

    def rotary(case, s):
        half = case["rotary_dim"] // 2
        first = torch.arange(half, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (half if case["layout"] == "half" else 1)
        out = []
        for name, turn in (("q", 1.0), ("k", 1.0), ("dq", -1.0), ("dk", -1.0)):
            if name not in s:
                continue
            x = s[name].detach()
            y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
            for b in range(case["batch"]):
                at = torch.arange(case["seq"], device="cuda") if s["pos"] is None else s["pos"][b].long()
                # The rotation as a complex product.
                angle = torch.complex(s["cos"][at].double(), turn * s["sin"][at].double())
                xb = x[b].double()
                z = torch.complex(xb[..., first], xb[..., second]) * angle
                y[b] = xb
                y[b][..., first], y[b][..., second] = z.real, z.imag
            out.append(y)
        return out

    def tree(case, s):
        group = case["q_heads"] // case["kv_heads"]
        out = torch.empty(case["batch"], case["q_heads"], case["tree"], case["dim"], dtype=torch.float64, device="cuda")
        parents = None if s["parents"] is None else s["parents"].tolist()
        for b in range(case["batch"]):
            n = int(s["lens"][b])
            seen = torch.zeros(case["tree"], n + case["tree"], dtype=torch.bool)
            seen[:, :n] = True
            for i in range(case["tree"]):
                node = i
                while node >= 0:
                    seen[i, n + node] = True
                    node = node - 1 if parents is None else parents[b][node]
            seen = seen.cuda()
            for h in range(case["kv_heads"]):
                keys = torch.cat((s["k_cache"][b, h, :n], s["k_tree"][b, h])).double()
                values = torch.cat((s["v_cache"][b, h, :n], s["v_tree"][b, h])).double()
                q = s["q"][b, h * group : (h + 1) * group].double()
                scores = torch.einsum("gtd,nd->gtn", q, keys) / math.sqrt(case["dim"])
                weights = torch.softmax(torch.where(seen, scores, float("-inf")), -1)
                out[b, h * group : (h + 1) * group] = weights @ values
        return out

    def verify(case, s):
        tree = case["tree"]
        path = torch.full((case["batch"], tree), -1, dtype=torch.int32)
        lengths, nexts = torch.zeros(case["batch"], dtype=torch.int32), torch.zeros(case["batch"], dtype=torch.int64)
        tokens, uniforms = s["tokens"].tolist(), s["uniforms"].double().tolist()
        parents = None if s["parents"] is None else s["parents"].tolist()
        for b in range(case["batch"]):
            node, walk = 0, [0]
            while True:
                p = s["target"][b, node].double()
                children = [c for c in range(1, tree) if (c - 1 if parents is None else parents[b][c]) == node]
                weights, found = p.clone(), None
                for c in children:
                    x = tokens[b][c]
                    if case["draft"]:
                        q = s["draft_probs"][b, node].double()
                        accepted = uniforms[b][c] * float(q[x]) < float(p[x])
                        weights = (p - q).clamp_min(0.0)
                    else:
                        mass = 1.0 - sum(float(p[t]) for t in {tokens[b][o] for o in children if o < c})
                        accepted = uniforms[b][c] * max(mass, 0.0) < float(weights[x])
                        weights[x] = 0.0
                    if accepted:
                        found = c
                        break
                if found is None:
                    break
                node = found
                walk.append(node)
            if float(weights.max()) <= 0.0:
                weights = p
            path[b, : len(walk)] = torch.tensor(walk, dtype=torch.int32)
            lengths[b], nexts[b] = len(walk), int((weights / s["noise"][b].double()).argmax())
        return [path, lengths, nexts]

    def commit(case, s):
        lens = s["lens"].clone()
        for name in ("k", "v"):
            for b in range(case["batch"]):
                n, start = int(s["path_lens"][b]), int(s["lens"][b])
                s[name + "_cache"][:, b, :, start : start + n] = s[name + "_tree"][:, b][:, :, s["path"][b, :n].long()]
                lens[b] = start + n
        return [s["k_cache"], s["v_cache"], lens]

    of = {"rotary": rotary, "tree": tree, "verify": verify, "commit": commit}
    with torch.no_grad():
        return of[case["op"]](case, prepare(case, seed))
