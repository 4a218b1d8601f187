"""``tklab.kernels.speculative``: verification and the cache commit against the references, and their refusals."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from oracle.speculative_oracle import commit_reference, verify_reference
from tklab import _native
from tklab._tensors import binding
from tklab.kernels.flash_attention import check_device_status
from tklab.kernels.speculative import commit_draft, verify_draft

gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU is required")


def trees(gen, batch, nodes):
    index = torch.arange(nodes)
    parents = torch.minimum((torch.rand(batch, nodes, generator=gen).sqrt() * index).floor(), (index - 1).clamp_min(0)).int()
    parents[:, 0] = -1
    return parents


def draft_of(batch, nodes, vocab, *, kind, dtype=torch.float32, seed=0, sharp=2.0):
    """Inputs whose drafts are drawn from the target ("tree", "chain") or a nearby draft model ("draft")."""
    gen = torch.Generator().manual_seed(seed)
    logits = sharp * torch.randn(batch, nodes, vocab, generator=gen)
    target = logits.softmax(-1).to(dtype)
    parents = trees(gen, batch, nodes) if kind == "tree" else None
    draft = None
    source = target
    if kind == "draft":
        draft = (logits[:, : nodes - 1] + 0.7 * torch.randn(batch, nodes - 1, vocab, generator=gen)).softmax(-1).to(dtype)
        source = draft
    tokens = torch.randint(0, vocab, (batch, nodes), generator=gen)
    for b in range(batch):
        for c in range(1, nodes):
            n = c - 1 if parents is None else int(parents[b, c])
            tokens[b, c] = int(torch.multinomial(source[b, n].float(), 1, generator=gen))
    return {
        "target_probs": target, "tokens": tokens, "uniforms": torch.rand(batch, nodes, generator=gen),
        "noise": torch.empty(batch, vocab).exponential_(generator=gen).clamp_min(1e-9), "parents": parents, "draft_probs": draft,
    }


def on_gpu(p):
    return {n: t.cuda() if torch.is_tensor(t) else t for n, t in p.items()}


def check(p, **kwargs):
    got = verify_draft(**on_gpu(p), **on_gpu(kwargs))
    want = verify_reference(p["target_probs"], p["tokens"], p["uniforms"], p["noise"], parents=p["parents"], draft=p["draft_probs"], **kwargs)
    for g, w in zip(got, want, strict=True):
        assert g.dtype == w.dtype and torch.equal(g.cpu(), w)
    check_device_status()
    return got


# ---------------------------------------------------------------- refusals
def test_verify_refuses() -> None:
    p = draft_of(2, 3, 10, kind="draft")

    def bad(match, **change):
        with pytest.raises(ValueError, match=match):
            verify_draft(**{**p, **change})

    bad("target_probs must be a non-empty", target_probs=p["target_probs"][0])
    bad("non-empty", target_probs=p["target_probs"][:, :, :0])
    bad("float32, bfloat16 or float16", target_probs=p["target_probs"].double())
    bad("tokens", tokens=p["tokens"].float())
    bad("tokens", tokens=p["tokens"][:, :2])
    bad("uniforms", uniforms=p["uniforms"].half())
    bad("noise", noise=p["noise"][:1])
    bad("chains only", parents=torch.tensor([-1, 0, 0], dtype=torch.int32))
    bad("nodes - 1", draft_probs=p["target_probs"])
    bad("CUDA")


@pytest.mark.parametrize(
    ("kwargs", "status"),
    [
        ({"target": None}, 1), ({"noise": None}, 1), ({"next": None}, 1), ({"batch": 0}, 1), ({"vocab": 0}, 1),
        ({"draft": 0x1000, "draft_strides": (ctypes.c_int64 * 2)(64, 8), "parents": 0x1000, "parent_stride": 4}, 1),
        ({"draft": 0x1000}, 1), ({"parents": 0x1000, "parent_stride": 3}, 1), ({"prob_type": 3}, 2),
        ({"nodes": 257}, 2), ({"target": 0x1002}, 3), ({"path": 0x1002}, 3), ({"tokens": 0x1004}, 3),
    ],
)
def test_library_verify_refuses_before_launch(kwargs: dict, status: int) -> None:
    args = {"target": 0x1000, "target_strides": (ctypes.c_int64 * 2)(64, 8), "draft": None, "draft_strides": None,
            "tokens": 0x1000, "tokens_64": 1, "parents": None, "parent_stride": 0, "tree_sizes": None, "uniforms": 0x1000,
            "noise": 0x1000, "path": 0x1000, "path_lens": 0x1000, "next": 0x1000, "batch": 1, "nodes": 4, "vocab": 8,
            "prob_type": 2, "stream": None}
    args.update(kwargs)
    assert _native.load().tk_verify_draft(*args.values()) == status


def test_commit_refuses() -> None:
    cache, tree = torch.zeros(2, 2, 8, 16, dtype=torch.float16), torch.zeros(2, 2, 3, 16, dtype=torch.float16)
    path, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)

    def bad(match, k=cache, v=cache, kt=tree, vt=tree):
        with pytest.raises(ValueError, match=match):
            commit_draft(k, v, kt, vt, path, lens, lens)

    bad("identical shapes", v=cache[:, :1])
    bad("identical shapes", k=cache[0], v=cache[0])
    bad("disagree", kt=tree[:, :1], vt=tree[:, :1])
    bad("empty", k=cache[:, :, :0], v=cache[:, :, :0])
    bad("dtype", k=cache.float(), v=cache.float())
    bad("CUDA")


@pytest.mark.parametrize(
    ("kwargs", "status"),
    [
        ({"k": None}, 1), ({"new_lens": 0x2000}, 1), ({"layers": 0}, 1), ({"nodes": 0}, 1), ({"head_dim": 12}, 2),
        ({"nodes": 300}, 2), ({"v_tree": 0x1008}, 3), ({"path": 0x1001}, 3), ({"strides": (ctypes.c_int64 * 16)(*[4] * 16)}, 3),
        ({"batch": 1 << 20}, 8),
    ],
)
def test_library_commit_refuses_before_launch(kwargs: dict, status: int) -> None:
    args = {"k": 0x1000, "v": 0x1000, "k_tree": 0x1000, "v_tree": 0x1000, "strides": (ctypes.c_int64 * 16)(*[64] * 16),
            "path": 0x1000, "path_lens": 0x1000, "kv_lens": 0x2000, "new_lens": 0x3000, "layers": 1, "batch": 1,
            "kv_heads": 1, "nodes": 3, "seq_kv": 8, "head_dim": 16, "stream": None}
    args.update(kwargs)
    assert _native.load().tk_commit_draft(*args.values()) == status


def test_overlap_of_trees_and_caches_is_found() -> None:
    """Against the sets of elements: views of one buffer in every order of dimensions, whole and in part, near and far."""
    gen = random.Random(1)
    apart = 0
    for _ in range(2000):
        sizes = [gen.randint(1, 4) for _ in range(3)] + [gen.randint(4, 9), 8]
        order = gen.sample(range(4), 4) + [4]
        buffer = torch.arange(math.prod(sizes), dtype=torch.int16).view([sizes[i] for i in order])
        whole = buffer.permute([order.index(i) for i in range(5)])
        views = []
        for _ in range(2):
            view = whole
            for axis in range(5):
                if gen.random() < (0.8 if axis == 3 else 0.3):
                    start = gen.randrange(sizes[axis])
                    view = view.narrow(axis, start, gen.randint(1, sizes[axis] - start))
            views.append(view)
        common = not set(views[0].flatten().tolist()).isdisjoint(views[1].flatten().tolist())
        assert binding.may_overlap(*views) == common
        apart += not common
    assert 200 < apart < 1800
    other = torch.arange(64, dtype=torch.int16)
    assert not binding.may_overlap(other[:32], other[32:].clone()) and binding.may_overlap(other[::2], other[1::3])  # not known


# ------------------------------------------------------------ verification
@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
@pytest.mark.parametrize(("nodes", "vocab"), [(1, 50), (2, 1), (5, 7), (6, 1001), (33, 257), (64, 4099)])
def test_verify_matches_reference(dtype: torch.dtype, kind: str, nodes: int, vocab: int) -> None:
    check(draft_of(9, nodes, vocab, kind=kind, dtype=dtype, seed=nodes + vocab))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_large_vocabularies_and_batches(kind: str) -> None:
    check(draft_of(3, 4, 100003, kind=kind, seed=5, sharp=4.0))
    check(draft_of(400, 3, 40, kind=kind, seed=6))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 6, 7, 9, 10, 11, 13, 509, 2050, 4101, 20483])
def test_verify_rows_that_start_anywhere(dtype: torch.dtype, vocab: int) -> None:
    """Rows of every alignment, in tensors that start and end anywhere in their storage; winners at both ends of a row."""
    p = draft_of(8, 3, vocab, kind="tree", dtype=dtype, seed=vocab)
    p["noise"][0::4, 0] = 1e-6
    p["noise"][1::4, -1] = 1e-6
    p["noise"][2::4, min(vocab - 1, 3)] = 1e-6
    ref = check(p)
    g = on_gpu(p)
    for before in range(4):
        target = torch.full((8 * 3 * vocab + before,), math.nan, dtype=dtype, device="cuda")[before:].view(8, 3, vocab)
        target.copy_(g["target_probs"])
        noise = torch.full((8 * vocab + 3 - before,), -1.0, device="cuda")[3 - before :].view(8, vocab)
        noise.copy_(g["noise"])
        padded = torch.full((8, 3, vocab + 5), math.nan, dtype=dtype, device="cuda")[..., before : before + vocab]
        padded.copy_(g["target_probs"])
        for change in ({"target_probs": target}, {"noise": noise}, {"target_probs": padded, "noise": noise}):
            for a, b in zip(ref, verify_draft(**{**g, **change}), strict=True):
                assert torch.equal(a, b)
    check_device_status()


@pytest.mark.gpu
@gpu
def test_verify_many_nodes_and_sizes() -> None:
    p = draft_of(6, 256, 90, kind="tree", seed=9, sharp=3.0)
    check(p, tree_sizes=torch.tensor([256, 0, 1, 100, -4, 900], dtype=torch.int32))
    p = draft_of(4, 256, 20, kind="chain", seed=10, sharp=3.0)
    p["uniforms"][1:] = 0.0  # everything that has any probability is accepted
    got = check(p)
    assert int(got.path_lens[2]) == 256


@pytest.mark.gpu
@gpu
def test_verify_duplicates_outsiders_and_ties() -> None:
    p = draft_of(1, 6, 4, kind="tree", seed=1)
    p["parents"] = torch.tensor([-1, 0, 0, 0, 0, 2], dtype=torch.int32)
    p["target_probs"][:] = 0.25
    p["uniforms"] = torch.tensor([[0.0, 0.3, 0.2, 0.9, 0.9, 0.1]])
    p["noise"][:] = 1.0
    for tokens in ([0, 1, 1, 1, 1, 2], [0, 1, 9, -3, 2, 2], [0, 3, 2, 1, 0, 3], [0, 0, 1, 2, 3, 3], [0, 2**40, 0, 0, 0, 0]):
        p["tokens"] = torch.tensor([tokens])
        check(p)
        check({**p, "uniforms": torch.full((1, 6), 0.999)})
    p["target_probs"] = torch.tensor([1.0, 0.0, 0.0, 0.0]).expand(1, 6, 4).contiguous()
    p["tokens"] = torch.tensor([[0, 0, 1, 2, 3, 0]])
    check({**p, "uniforms": torch.full((1, 6), 0.999)})
    # Draft and target equal: nothing is left after a refusal, the target itself is drawn from.
    q = draft_of(1, 2, 8, kind="draft", seed=3)
    q["target_probs"][:, 0] = q["draft_probs"][:, 0]
    q["tokens"][0, 1] = 5
    check({**q, "uniforms": torch.ones(1, 2)})


@pytest.mark.gpu
@gpu
def test_verify_strides_types_and_nan() -> None:
    p = draft_of(5, 7, 130, kind="tree", seed=4)
    ref = check(p)
    g = on_gpu(p)
    for target in (
        g["target_probs"].transpose(0, 1).contiguous().transpose(0, 1),
        torch.nn.functional.pad(g["target_probs"], (1, 2))[..., 1:131],
        g["target_probs"].transpose(1, 2).contiguous().transpose(1, 2),
    ):
        for a, b in zip(ref, verify_draft(**{**g, "target_probs": target}), strict=True):
            assert torch.equal(a, b)
    narrow = verify_draft(**{**g, "tokens": g["tokens"].int()})
    assert narrow.next_tokens.dtype == torch.int32 and torch.equal(narrow.next_tokens.long(), ref.next_tokens)
    one = verify_draft(**{**g, "parents": g["parents"][0]})
    same = verify_draft(**{**g, "parents": g["parents"][:1].expand(5, 7)})
    for a, b in zip(one, same, strict=True):
        assert torch.equal(a, b)
    p["target_probs"][:, :, 3:50] = math.nan
    check(p)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = verify_draft(**g)
    side.synchronize()
    for a, b in zip(ref, got, strict=True):
        assert torch.equal(a, b)


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_emitted_tokens_follow_the_target(kind: str) -> None:
    """First emitted token of many independent steps: each frequency within five standard deviations of the target's."""
    n, vocab = 200_000, 6
    gen = torch.Generator(device="cuda").manual_seed(7)
    target = torch.tensor([[0.35, 0.3, 0.2, 0.1, 0.05, 0.0]], device="cuda").expand(n, vocab)
    other = torch.full((n, vocab), 1.0 / vocab, device="cuda")
    rand = lambda nodes: torch.rand(n, nodes, generator=gen, device="cuda")  # noqa: E731
    noise = torch.empty(n, vocab, device="cuda").exponential_(generator=gen)
    if kind == "draft":
        q = torch.tensor([0.1, 0.1, 0.2, 0.2, 0.2, 0.2], device="cuda")
        tokens = torch.zeros(n, 2, dtype=torch.int64, device="cuda")
        tokens[:, 1] = torch.multinomial(q, n, replacement=True, generator=gen)
        got = verify_draft(torch.stack((target, other), 1), tokens, rand(2), noise, draft_probs=q.expand(n, 1, vocab))
    else:
        tokens = torch.tensor([[0, 1, 3, 3, 0]], device="cuda").expand(n, 5)
        parents = torch.tensor([-1, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
        got = verify_draft(torch.stack((target, other, other, other, other), 1), tokens, rand(5), noise, parents=parents)
    first = torch.where(got.path_lens > 1, tokens.gather(1, got.path[:, 1:2].clamp_min(0).long())[:, 0], got.next_tokens)
    share = torch.bincount(first, minlength=vocab).double().cpu() / n
    p = target[0].double().cpu()
    assert bool(((share - p).abs() <= 5.0 * (p * (1.0 - p) / n).sqrt()).all()), share


# ------------------------------------------------------------------ commit
def commit_problem(layers, batch, heads, nodes, capacity, dim, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda rows: torch.randn(layers, batch, heads, rows, dim, generator=gen).to(dtype)  # noqa: E731
    length = torch.randint(1, nodes + 1, (batch,), generator=gen)
    path = torch.full((batch, nodes), -1, dtype=torch.int32)
    for b in range(batch):
        n = int(length[b])
        path[b, :n] = torch.cat((torch.zeros(1), 1 + torch.randperm(nodes - 1, generator=gen)[: n - 1].sort().values)).int()
    lens = torch.randint(0, capacity - nodes + 1, (batch,), generator=gen, dtype=torch.int32)
    return [rand(capacity), rand(capacity), rand(nodes), rand(nodes), path, length.int(), lens]


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(
    ("layers", "batch", "heads", "nodes", "capacity", "dim"),
    [(1, 1, 1, 1, 1, 8), (1, 3, 2, 5, 5, 64), (4, 3, 2, 9, 40, 128), (2, 5, 3, 64, 100, 72), (3, 2, 8, 256, 300, 16)],
)
def test_commit_matches_reference(layers, batch, heads, nodes, capacity, dim, dtype) -> None:
    args = commit_problem(layers, batch, heads, nodes, capacity, dim, dtype, seed=nodes)
    want = commit_reference(*args)
    gpu_args = [t.cuda() for t in args]
    lens = commit_draft(*gpu_args)
    for got, ref in zip((gpu_args[0], gpu_args[1], lens), want, strict=True):
        assert got.dtype == ref.dtype and torch.equal(got.cpu(), ref)
    assert torch.equal(gpu_args[6].cpu(), args[6])
    # Layer by layer, and from (batch, rows, heads, dim) storage.
    again = [t.cuda() for t in args]
    again[0] = again[0].transpose(2, 3).contiguous().transpose(2, 3)
    again[3] = again[3].transpose(2, 3).contiguous().transpose(2, 3)
    for i in range(layers):
        assert torch.equal(commit_draft(*(t[i] for t in again[:4]), *again[4:]), lens)
    assert torch.equal(again[0].cpu(), want[0]) and torch.equal(again[1].cpu(), want[1])
    check_device_status()


@pytest.mark.gpu
@gpu
def test_commit_into_a_full_cache_and_bad_paths() -> None:
    args = commit_problem(2, 3, 2, 6, 20, 64, torch.bfloat16, seed=2)
    args[5] = torch.tensor([6, 6, 0], dtype=torch.int32)
    args[4] = torch.arange(6, dtype=torch.int32).expand(3, 6).contiguous()
    args[6] = torch.tensor([17, 20, 4], dtype=torch.int32)
    want = commit_reference(*args)
    g = [t.cuda() for t in args]
    lens = commit_draft(*g)
    assert lens.tolist() == [20, 20, 4]
    assert torch.equal(g[0].cpu(), want[0]) and torch.equal(g[1].cpu(), want[1])
    with pytest.raises(RuntimeError, match="exceeds"):
        check_device_status()
    args[6], args[5] = torch.zeros(3, dtype=torch.int32), torch.full((3,), 2, dtype=torch.int32)
    args[4][:, 1] = torch.tensor([-1, 6, 2**30], dtype=torch.int32)
    g = [t.cuda() for t in args]
    before = g[0].clone()
    commit_draft(*g)
    with pytest.raises(RuntimeError, match="invalid argument"):
        check_device_status()
    assert torch.equal(g[0][:, :, :, 1:], before[:, :, :, 1:])
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("which", [0, 3])
def test_commit_of_a_tangent_is_an_error(which: int) -> None:
    g = [t.cuda() for t in commit_problem(1, 2, 2, 5, 20, 64, torch.bfloat16, seed=4)]
    with torch.autograd.forward_ad.dual_level():
        g[which] = torch.autograd.forward_ad.make_dual(g[which], torch.ones_like(g[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            commit_draft(*g)


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("which", [0, 1])
def test_commit_is_a_change_in_place(which: int) -> None:
    """What autograd saved of a cache before is known to be stale after, a view of one layer included."""
    for layers in (False, True):
        g = [t.cuda() for t in commit_problem(2, 2, 2, 5, 20, 64, torch.bfloat16, seed=5)]
        x = torch.ones((), device="cuda", requires_grad=True)
        loss = (x * g[which].float().mul_(1.0)).sum() + (x.bfloat16() * g[which]).sum()
        before = g[which]._version
        if layers:
            commit_draft(*g)
        else:
            commit_draft(*(t[1] for t in g[:4]), *g[4:])
        assert g[which]._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        g = [t.cuda() for t in commit_problem(1, 2, 2, 5, 20, 64, torch.bfloat16, seed=5)]
        want = commit_reference(*(t.cpu() for t in g))
        commit_draft(*g)
        assert torch.equal(g[0].cpu(), want[0]) and torch.equal(g[1].cpu(), want[1])
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(
    ("path_len", "kv_len", "rows", "start", "match"),
    [(7, 3, 6, 3, "invalid argument"), (-1, 3, 0, 3, "invalid argument"), (2, -4, 2, 0, "invalid argument"),
     (0, 21, 0, 20, "invalid argument"), (2, 21, 0, 20, "exceeds"), (6, 14, 6, 14, None), (0, 20, 0, 20, None)],
)
def test_commit_reports_lengths_that_it_clamps(path_len: int, kv_len: int, rows: int, start: int, match: str | None) -> None:
    args = [t.cuda() for t in commit_problem(2, 2, 3, 6, 20, 64, torch.float16, seed=8)]
    args[4] = torch.arange(6, dtype=torch.int32, device="cuda").expand(2, 6).contiguous()
    args[5], args[6] = (torch.tensor([n, 1], dtype=torch.int32, device="cuda") for n in (path_len, kv_len))
    want = args[0].clone()
    want[:, 0, :, start : start + rows] = args[2][:, 0, :, :rows]
    want[:, 1, :, 1] = args[2][:, 1, :, 0]
    assert commit_draft(*args).tolist() == [start + rows, 2]
    assert torch.equal(args[0], want)
    if match is not None:
        with pytest.raises(RuntimeError, match=match):
            check_device_status()
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("layers", [1, 3])
def test_commit_of_drafts_kept_in_the_cache(layers: int) -> None:
    """Trees that are rows of the caches, before, behind and among those written: copied as they were before the call."""
    for which in range(4):
        args = [t.cuda() for t in commit_problem(layers, 4, 3, 9, 40, 64, torch.bfloat16, seed=9)]
        args[4] = torch.tensor([[0, 2, 3, 5, 8, -1, -1, -1, -1]] * 4, dtype=torch.int32, device="cuda")
        args[5] = torch.tensor([5, 4, 5, 1], dtype=torch.int32, device="cuda")
        args[6] = torch.tensor([10, 12, 8, 15], dtype=torch.int32, device="cuda")
        if which in (0, 2):
            args[2] = args[0][:, :, :, 10:19]
        if which in (1, 2):
            args[3] = args[1][:, :, :, 10:19]
        if which == 3:
            args[2], args[3] = args[1][:, :, :, 9:18], args[0][..., 11:20, :]
        want = commit_reference(*(t.cpu() for t in args))
        if layers == 1:
            lens = commit_draft(*(t[0] for t in args[:4]), *args[4:])
        else:
            lens = commit_draft(*args)
        for got, ref in zip((args[0], args[1], lens), want, strict=True):
            assert torch.equal(got.cpu(), ref)
    check_device_status()


@pytest.mark.gpu
@gpu
def test_commit_copies_no_tree_beside_the_cache() -> None:
    """Trees in the caches' memory but apart from them (rows behind them, keys and values side by side) are read in place."""
    for layout in range(3):
        args = [t.cuda() for t in commit_problem(2, 3, 2, 6, 20, 64, torch.float16, seed=10)]
        want = commit_reference(*(t.cpu() for t in args))
        if layout == 0:
            for cache, tree in ((0, 2), (1, 3)):
                both = torch.cat((args[cache], args[tree]), 3)
                args[cache], args[tree] = both[:, :, :, :20], both[:, :, :, 20:]
        elif layout == 1:
            for cache, tree in ((0, 2), (1, 3)):
                both = torch.cat((args[cache], args[tree]), 3).transpose(2, 3).contiguous().transpose(2, 3)
                args[cache], args[tree] = both[:, :, :, :20], both[:, :, :, 20:]
        else:
            both = torch.stack((torch.cat((args[0], args[2]), 3), torch.cat((args[1], args[3]), 3)), 4)
            args[0], args[1] = both[:, :, :, :20, 0], both[:, :, :, :20, 1]
            args[2], args[3] = both[:, :, :, 20:, 0], both[:, :, :, 20:, 1]
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        lens = commit_draft(*args)
        assert torch.cuda.memory_stats()["allocation.all.allocated"] == before + 1  # the new lengths
        for got, ref in zip((args[0], args[1], lens), want, strict=True):
            assert torch.equal(got.cpu(), ref)
    check_device_status()
