"""``tklab.kernels.tree_attention`` against the 64-bit reference (GPU), and its refusals (CPU)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import load_selftest_lib
from oracle.speculative_oracle import tree_attention_reference
from tklab import _native
from tklab.kernels.flash_attention import check_device_status
from tklab.kernels.gqa_decode import gqa_decode
from tklab.kernels.tree_attention import tree_attention

gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU is required")
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def problem(batch, q_heads, kv_heads, nodes, dim, capacity, lens, dtype, *, seed=0, tree=True, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen).to(dtype)  # noqa: E731
    parents = None
    if tree:
        index = torch.arange(nodes)
        parents = torch.minimum((torch.rand(batch, nodes, generator=gen).sqrt() * index).floor(), (index - 1).clamp_min(0)).int()
        parents[:, 0] = -1
    return {
        "q": (spread * rand(batch, q_heads, nodes, dim)).to(dtype),
        "k_cache": rand(batch, kv_heads, capacity, dim), "v_cache": rand(batch, kv_heads, capacity, dim),
        "k_tree": rand(batch, kv_heads, nodes, dim), "v_tree": rand(batch, kv_heads, nodes, dim),
        "kv_lens": torch.tensor(lens, dtype=torch.int32), "parents": parents,
    }


def on_gpu(p):
    return {n: None if t is None else t.cuda() for n, t in p.items()}


def assert_attends(o, lse, ref):
    """P and o are rounded to the 16-bit type once each; the fp32 arithmetic (scores, exponentials, sums) stays below
    2^-12 of the weighted magnitude at these sizes; 16-bit P below 2^-14 (float16) adds 2^-25 a key at most."""
    ref_o, ref_lse, spread = ref
    bound = (2.0 * ROUND[o.dtype] + 2.0**-12) * spread + 2.0**-14 * 2.0**-3
    err = (o.double().cpu() - ref_o).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    if lse is not None:
        empty = torch.isinf(ref_lse)
        assert torch.equal(torch.isinf(lse.cpu()), empty) and bool((lse.cpu()[empty] < 0).all())
        off = (lse.double().cpu() - ref_lse)[~empty].abs()
        assert not off.numel() or float((off - 1e-6 * ref_lse[~empty].abs()).max()) <= 2e-4


def check(p, **kwargs):
    o, lse = tree_attention(**on_gpu(p), return_lse=True, **{n: v.cuda() if torch.is_tensor(v) else v for n, v in kwargs.items()})
    assert o.shape == p["q"].shape and o.dtype == p["q"].dtype
    assert_attends(o, lse, tree_attention_reference(**p, **kwargs))
    check_device_status()
    return o, lse


# ---------------------------------------------------------------- refusals
def test_refuses_bad_arguments() -> None:
    p = problem(2, 4, 2, 3, 64, 16, [4, 5], torch.float16)

    def bad(match, **change):
        with pytest.raises(ValueError, match=match):
            tree_attention(**{**p, **change})

    bad("4-dimensional", q=p["q"][0])
    bad("identical", v_cache=p["v_cache"][:, :1])
    bad("the tree's", k_tree=p["k_tree"][:, :, :2])
    bad("empty", q=p["q"][:, :, :0], k_tree=p["k_tree"][:, :, :0], v_tree=p["v_tree"][:, :, :0])
    bad("multiple of kv_heads", q=p["q"][:, :3])
    bad("share one dtype", q=p["q"].float())
    bad("share one dtype", v_tree=p["v_tree"].bfloat16())
    bad("CUDA")
    big = problem(1, 1, 1, 257, 8, 8, [1], torch.float16)
    with pytest.raises(ValueError, match="256 nodes"):
        tree_attention(**big)
    wide = problem(1, 1, 1, 2, 136, 8, [1], torch.float16)
    with pytest.raises(ValueError, match="head_dim"):
        tree_attention(**wide)


@pytest.mark.parametrize(
    ("kwargs", "status"),
    [
        ({"q": None}, 1), ({"kv_lens": None}, 1), ({"strides": None}, 1), ({"batch": 0}, 1), ({"q_heads": 3}, 1),
        ({"nodes": 0}, 1), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"parent_stride": 2}, 1),
        ({"head_dim": 20}, 2), ({"head_dim": 136}, 2), ({"nodes": 257, "parent_stride": 257}, 2), ({"dtype": 3}, 2),
        ({"o": 0x1008}, 3), ({"lse": 0x1002}, 3), ({"kv_lens": 0x1001}, 3), ({"workspace": 0x1010}, 3),
        ({"seq_kv": 1 << 31}, 8),
    ],
)
def test_library_refuses_before_launch(kwargs: dict, status: int) -> None:
    args = {"q": 0x1000, "k": 0x1000, "v": 0x1000, "k_tree": 0x1000, "v_tree": 0x1000,
            "strides": (ctypes.c_int64 * 12)(*[64] * 12), "kv_lens": 0x1000, "parents": 0x1000, "parent_stride": 3,
            "tree_sizes": None, "o": 0x1000, "lse": None, "workspace": None, "workspace_bytes": 0, "batch": 1,
            "q_heads": 4, "kv_heads": 2, "nodes": 3, "seq_kv": 16, "head_dim": 64, "dtype": 1, "scale": 0.125,
            "stream": None}
    args.update(kwargs)
    assert _native.load().tk_tree_attn(*args.values()) == status


def test_joining_takes_entries_of_cut_items_only() -> None:
    """Whatever an entry holds where a CTA gave up, no part past the runs' and no row past the items' is touched."""
    ok = load_selftest_lib().tk_selftest_tree_cut_ok
    big = 2**31 - 1
    for item, run, slot, parts, good in [
        (0, 0, 0, 1, 1), (11, 0, 1, 148, 1), (5, 147, 1, 1, 1), (-1, 0, 0, 0, 0), (12, 0, 0, 1, 0), (0, 148, 0, 1, 0),
        (0, -1, 0, 1, 0), (0, 0, 2, 1, 0), (0, 0, -1, 1, 0), (0, 0, 0, 0, 0), (0, 0, 0, 149, 0), (0, 147, 0, 2, 0),
        (big, big, big, big, 0), (0, big, 0, 1, 0), (0, 1, 0, big, 0), (-big, -big, -big, -big, 0), (0, 0, 0, -big, 0),
    ]:
        assert ok(item, run, slot, parts, 12, 148) == good, (item, run, slot, parts)


# --------------------------------------------------------------------- GPU

@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
@pytest.mark.parametrize("nodes", [1, 2, 7, 16, 33, 64])
def test_matches_reference(dtype: torch.dtype, dim: int, group: int, nodes: int) -> None:
    lens = [0, 1, 127, 128, 129, 300]
    check(problem(6, 2 * group, 2, nodes, dim, 301, lens, dtype, seed=nodes + group))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 96, 120])
def test_odd_head_dims(dim: int) -> None:
    check(problem(2, 6, 2, 11, dim, 200, [150, 64], torch.bfloat16, seed=dim))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("group", "nodes"), [(1, 127), (1, 128), (1, 129), (2, 200), (3, 256), (16, 33), (16, 40), (5, 77)])
@pytest.mark.parametrize("tree", [False, True])
def test_many_rows(group: int, nodes: int, tree: bool) -> None:
    """More rows than one tile of 128, trees of more than one tile, chains and trees."""
    check(problem(2, group, 1, nodes, 64, 400, [400, 77], torch.float16, seed=nodes, tree=tree))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(("batch", "capacity", "nodes"), [(1, 5000, 5), (3, 3333, 20), (1, 20000, 1)])
def test_split_lengths(dim: int, batch: int, capacity: int, nodes: int) -> None:
    """Long caches, split over many CTAs; scores that grow along the cache move the running maxima."""
    lens = [capacity, capacity // 3, 1][:batch]
    p = problem(batch, 8, 2, nodes, dim, capacity, lens, torch.bfloat16, seed=capacity)
    p["k_cache"] = (p["k_cache"].float() * torch.linspace(0.1, 2.5, capacity)[None, None, :, None]).bfloat16()
    o, lse = check(p)
    o2, lse2 = tree_attention(**on_gpu(p), return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)  # the same bits every time


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("batch", [40, 200])
def test_many_sequences_of_mixed_length(batch: int) -> None:
    lens = [(37 * i * i + 11) % 601 for i in range(batch)]
    check(problem(batch, 4, 2, 6, 64, 600, lens, torch.bfloat16, seed=batch))  # one length above the capacity's use, some 0


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_unused_rows_may_hold_anything(bad: float, dim: int) -> None:
    p = problem(4, 8, 2, 9, dim, 300, [300, 150, 0, 129], torch.bfloat16, seed=3)
    sizes = torch.tensor([9, 4, 1, 0], dtype=torch.int32)
    clean = check(p, tree_sizes=sizes)
    for b in range(4):
        for name in ("k", "v"):
            p[name + "_cache"][b, :, int(p["kv_lens"][b]) :] = bad
            p[name + "_tree"][b, :, int(sizes[b]) :] = bad
        p["q"][b, :, int(sizes[b]) :] = bad
    dirty = tree_attention(**on_gpu(p), tree_sizes=sizes.cuda(), return_lse=True)
    for a, b in zip(clean, dirty, strict=True):
        assert torch.equal(a, b)
    assert bool((dirty[0][3] == 0).all()) and bool((dirty[0][1, :, 4:] == 0).all())
    check_device_status()


@pytest.mark.gpu
@gpu
def test_lengths_past_the_cache_and_below_zero_are_clamped() -> None:
    p = problem(2, 4, 2, 3, 64, 100, [100, 0], torch.float16, seed=8)
    o = tree_attention(**on_gpu(p))
    p["kv_lens"] = torch.tensor([1000, -5], dtype=torch.int32)
    assert torch.equal(o, tree_attention(**on_gpu(p)))
    full = torch.tensor([99, -1], dtype=torch.int32)
    o = tree_attention(**on_gpu(p), tree_sizes=full.cuda())
    assert torch.equal(o, tree_attention(**on_gpu(p), tree_sizes=full.clamp(0, 3).cuda()))
    check_device_status()


@pytest.mark.gpu
@gpu
def test_parents_forms() -> None:
    """A chain given as parents, one tree for the batch, several roots, parents that are none."""
    p = problem(3, 4, 2, 12, 64, 90, [90, 10, 33], torch.bfloat16, seed=4, tree=False)
    o = tree_attention(**on_gpu(p))
    chain = torch.arange(-1, 11, dtype=torch.int32)
    assert torch.equal(o, tree_attention(**on_gpu({**p, "parents": chain})))
    assert torch.equal(o, tree_attention(**on_gpu({**p, "parents": chain.expand(3, 12)})))
    odd = torch.tensor([-1, -1, 0, 1, 9, 5, 2, -7, 3, 3, 2**30, 10], dtype=torch.int32)
    check({**p, "parents": odd})


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strided_caches_and_trees(dtype: torch.dtype) -> None:
    p = problem(3, 8, 4, 5, 64, 70, [70, 1, 40], dtype, seed=12)
    ref = tree_attention(**on_gpu(p))
    g = on_gpu(p)
    # (batch, rows, heads, dim) storage seen as (batch, heads, rows, dim); K and V interleaved; padded rows.
    bshd = {n: g[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("k_cache", "v_cache", "k_tree", "v_tree")}
    assert torch.equal(ref, tree_attention(**{**g, **bshd}))
    both = torch.stack((g["k_cache"], g["v_cache"]), 2)
    assert torch.equal(ref, tree_attention(**{**g, "k_cache": both[:, :, 0], "v_cache": both[:, :, 1]}))
    padded = torch.nn.functional.pad(g["v_cache"], (8, 16))[..., 8:72]
    assert torch.equal(ref, tree_attention(**{**g, "v_cache": padded}))
    odd = torch.nn.functional.pad(g["k_tree"], (1, 2))[..., 1:65]
    assert torch.equal(ref, tree_attention(**{**g, "k_tree": odd, "q": torch.nn.functional.pad(g["q"], (3, 0))[..., 3:]}))
    with pytest.raises(ValueError, match="the K cache"):
        tree_attention(**{**g, "k_cache": torch.nn.functional.pad(g["k_cache"], (1, 2))[..., 1:65]})
    with pytest.raises(ValueError, match="the V cache"):
        tree_attention(**{**g, "v_cache": g["v_cache"][:, :1].expand(3, 4, 70, 64)})
    check_device_status()


@pytest.mark.gpu
@gpu
def test_one_node_equals_decode_of_the_extended_cache() -> None:
    p = on_gpu(problem(2, 16, 4, 1, 128, 500, [400, 77], torch.bfloat16, seed=2))
    o, lse = tree_attention(**p, return_lse=True)
    for b, n in enumerate((400, 77)):
        p["k_cache"][b, :, n], p["v_cache"][b, :, n] = p["k_tree"][b, :, 0], p["v_tree"][b, :, 0]
    o2, lse2 = gqa_decode(p["q"], p["k_cache"], p["v_cache"], kv_lens=p["kv_lens"] + 1, return_lse=True)
    assert (o.float() - o2.float()).abs().max().item() <= 1e-2
    assert torch.allclose(lse[:, :, 0], lse2, atol=1e-3)
    check_device_status()


@pytest.mark.gpu
@gpu
def test_scale_large_scores_and_other_streams() -> None:
    p = problem(2, 4, 2, 6, 64, 333, [333, 200], torch.float16, seed=15, spread=6.0)
    check(p, scale=0.3)
    g = on_gpu(p)
    ref = tree_attention(**g, scale=0.3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o = tree_attention(**g, scale=0.3)
    side.synchronize()
    assert torch.equal(o, ref)


@pytest.mark.gpu
@gpu
def test_rows_past_32_bit_offsets() -> None:
    """The last rows of a cache of more than 2^31 elements."""
    capacity, dim = 2**31 // 128 // 2 + 1000, 128
    cache = torch.zeros(1, 2, capacity, dim, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    last = torch.randn(500, dim, generator=gen, device="cuda").bfloat16()
    cache[0, 1, -500:] = last
    view = cache[:, 1:, :]  # starts past 2^30 elements
    whole = torch.cat((cache[:, 1:, :1], cache[:, 1:, -500:]), 2)
    q = torch.randn(1, 2, 3, dim, generator=gen, device="cuda").bfloat16()
    tree = torch.randn(1, 1, 3, dim, generator=gen, device="cuda").bfloat16()
    lens = torch.tensor([capacity], dtype=torch.int32, device="cuda")
    # Zero keys score 0 and carry zero values: they only add their count to the sum.
    o, lse = tree_attention(q, view, view, tree, tree, lens, return_lse=True)
    zeros = capacity - 501
    ref_o, ref_lse, _ = tree_attention_reference(q.cpu(), whole.cpu(), whole.cpu(), tree.cpu(), tree.cpu(), torch.tensor([501]))
    total = torch.exp2(ref_lse) + zeros
    assert torch.allclose(lse.double().cpu(), torch.log2(total), atol=1e-3)
    expect = ref_o * (torch.exp2(ref_lse) / total)[..., None]
    assert (o.double().cpu() - expect).abs().max().item() <= 2.0**-7 * float(expect.abs().max()) + 1e-6
    both = tree_attention(q.repeat(1, 2, 1, 1), cache, cache, tree.repeat(1, 2, 1, 1), tree.repeat(1, 2, 1, 1), lens)
    assert torch.equal(both[:, 2:], o)
    check_device_status()


# Rows of one KV head (group x nodes) for every number of copies and tiles of the rows: up to 32, 64, 128, 256 and beyond.
ROWS = [(1, 1), (4, 8), (3, 11), (8, 8), (5, 13), (8, 16), (3, 43), (8, 32), (1, 200), (5, 77)]


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(("group", "nodes"), ROWS)
def test_items_cut_between_ctas(dtype: torch.dtype, dim: int, group: int, nodes: int) -> None:
    """Caches long enough that a sequence is shared by several CTAs, beside one of a few keys and an empty one."""
    p = problem(4, 2 * group, 2, nodes, dim, 2600, [2600, 0, 1025, 3], dtype, seed=group + nodes)
    sizes = torch.tensor([nodes, nodes, max(nodes - 3, 0), nodes // 2], dtype=torch.int32)
    o, lse = check(p, tree_sizes=sizes)
    o2, lse2 = tree_attention(**on_gpu(p), tree_sizes=sizes.cuda(), return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
@pytest.mark.parametrize(("group", "nodes"), ROWS[1::2])
def test_unused_rows_of_cut_items_may_hold_anything(bad: float, group: int, nodes: int) -> None:
    p = problem(3, 2 * group, 2, nodes, 128, 1500, [1400, 0, 515], torch.bfloat16, seed=nodes)
    sizes = torch.tensor([nodes // 2, nodes, 0], dtype=torch.int32)
    clean = check(p, tree_sizes=sizes)
    for b in range(3):
        for name in ("k", "v"):
            p[name + "_cache"][b, :, int(p["kv_lens"][b]) :] = bad
            p[name + "_tree"][b, :, int(sizes[b]) :] = bad
        p["q"][b, :, int(sizes[b]) :] = bad
    dirty = tree_attention(**on_gpu(p), tree_sizes=sizes.cuda(), return_lse=True)
    for a, b in zip(clean, dirty, strict=True):
        assert torch.equal(a, b)
    assert bool((dirty[0][2] == 0).all()) and bool(torch.isinf(dirty[1][2]).all())
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("group", "nodes"), [(2, 16), (4, 16), (8, 16), (8, 32)])
def test_more_sequences_than_ctas(group: int, nodes: int) -> None:
    """Runs of many short items: whole ones inside a run, cut ones at its ends, empty ones between them."""
    lens = [(53 * i * i + 7 * i) % 400 if i % 5 else 0 for i in range(130)]
    p = problem(130, 2 * group, 2, nodes, 64, 400, lens, torch.bfloat16, seed=nodes)
    check(p, tree_sizes=torch.tensor([(3 * i) % (nodes + 1) for i in range(130)], dtype=torch.int32))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("nodes", [5, 40])
def test_infinite_cache_rows_in_use(nodes: int) -> None:
    """An infinite key makes NaN of the rows whose score it makes +inf or NaN, as the formula does, and of no others."""
    p = problem(2, 4, 2, nodes, 64, 1300, [1300, 1300], torch.float16, seed=6)
    ref = tree_attention(**on_gpu(p))
    p["k_cache"][0, 1, 700] = math.inf
    o = tree_attention(**on_gpu(p))
    assert bool(torch.isnan(o[0, 2:]).all())
    assert torch.equal(o[0, :2], ref[0, :2]) and torch.equal(o[1], ref[1])
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("capacity", "nodes"), [(1300, 5), (1300, 20), (1300, 40), (1300, 100), (200, 5), (200, 100)])
def test_nan_query_rows_stay_nan(capacity: int, nodes: int) -> None:
    """A query of NaN has NaN for its output, and no other row does: cut items and items of one CTA."""
    p = problem(2, 4, 2, nodes, 64, capacity, [capacity, capacity // 3], torch.bfloat16, seed=9)
    ref = tree_attention(**on_gpu(p))
    p["q"][0, 1, nodes - 1, 3] = math.nan
    o, lse = tree_attention(**on_gpu(p), return_lse=True)
    assert bool(torch.isnan(o[0, 1, nodes - 1]).all()) and bool(torch.isnan(lse[0, 1, nodes - 1]))
    o[0, 1, nodes - 1] = ref[0, 1, nodes - 1]
    assert torch.equal(o, ref)
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("group", "capacity"), [(80, 1500), (80, 200), (160, 1400)])
def test_more_groups_of_rows_than_runs(group: int, capacity: int) -> None:
    """Rows in so many groups that each has one run, and in more groups than the device has SMs."""
    check(problem(2, group, 1, 256, 64, capacity, [capacity, 130], torch.bfloat16, seed=group))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("group", "nodes"), [(1, 1), (4, 8), (3, 11), (8, 8), (8, 16)])
@pytest.mark.parametrize("capacity", [300, 1300, 2600])
def test_nan_key_beside_large_scores(group: int, nodes: int, capacity: int) -> None:
    """Scores of some hundreds: whatever part of a row has the NaN weighs nothing beside the others, and the row is NaN."""
    p = problem(2, 2 * group, 2, nodes, 64, capacity, [capacity, capacity // 2], torch.bfloat16, seed=nodes, spread=100.0)
    ref = tree_attention(**on_gpu(p))
    p["k_cache"][0, 1, 140] = math.nan
    o, lse = tree_attention(**on_gpu(p), return_lse=True)
    assert bool(torch.isnan(o[0, group:]).all()) and bool(torch.isnan(lse[0, group:]).all())
    assert torch.equal(o[0, :group], ref[0, :group]) and torch.equal(o[1], ref[1])
    check_device_status()


def assert_attends_like(o, lse, ref):
    """:func:`assert_attends` where the formula is finite; the same infinities and NaN where it is not (of the
    log-sum-exp: none that is finite, for a score of +inf makes it +inf and the kernel's NaN)."""
    ref_o, ref_lse, spread = ref
    got, got_lse = o.double().cpu(), lse.double().cpu()
    odd = ~torch.isfinite(ref_o)
    assert torch.equal(torch.nan_to_num(got[odd], nan=0.0), torch.nan_to_num(ref_o[odd], nan=0.0))
    lost = torch.isnan(ref_lse) | (ref_lse == math.inf)
    assert torch.equal(torch.isnan(got), torch.isnan(ref_o)) and torch.equal(torch.isnan(got_lse) | (got_lse == math.inf), lost)
    put = lambda x, at: torch.where(at, torch.zeros_like(x), x)  # noqa: E731
    assert_attends(put(got, odd).to(o.dtype), put(got_lse, lost).float(), (put(ref_o, odd), put(ref_lse, lost), put(spread, odd)))


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(("group", "nodes"), [(3, 11), (8, 8), (3, 43), (8, 32)])
@pytest.mark.parametrize("capacity", [300, 1800])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_keys_that_are_not_finite_count_at_every_column(dtype, dim, group, nodes, capacity, bad) -> None:
    """One entry of a key, at eight columns of a whole tile, items of one CTA and cut ones: a score of NaN or +inf makes
    NaN of its row as the formula does, whatever the rows' number, and one of -inf takes the key out."""
    p = problem(8, group, 1, nodes, dim, capacity, [capacity] * 8, dtype, seed=dim + nodes)
    for b, column in enumerate((0, 3, 4, 7, 8, 11, 12, 15)):
        p["k_cache"][b, 0, 128 + column, 5] = bad
    o, lse = tree_attention(**on_gpu(p), return_lse=True)
    assert_attends_like(o, lse, tree_attention_reference(**p))
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 120])
@pytest.mark.parametrize(("group", "nodes"), ROWS[1:])
@pytest.mark.parametrize("capacity", [200, 1500])
@pytest.mark.parametrize("tree", [False, True])
def test_values_of_other_nodes_may_hold_anything(dtype, dim, group, nodes, capacity, tree) -> None:
    """Entries of drafted values that are not finite reach the nodes that attend them, as the formula has it, and no others."""
    p = problem(3, 2 * group, 2, nodes, dim, capacity, [capacity, 0, 77], dtype, seed=nodes + dim, tree=tree)
    clean = tree_attention(**on_gpu(p), return_lse=True)
    for b in range(3):
        for h in range(2):
            at = torch.randperm(nodes, generator=torch.Generator().manual_seed(2 * b + h))[: 3 if nodes > 3 else 1].tolist()
            for node, bad, column in zip(at, (math.nan, math.inf, -math.inf), (5, dim - 1, 8), strict=False):
                p["v_tree"][b, h, node, column] = bad
    p["v_tree"][2, 1, nodes - 1] = math.nan
    o, lse = tree_attention(**on_gpu(p), return_lse=True)
    ref_o = tree_attention_reference(**p)[0]
    fine = torch.isfinite(ref_o).cuda()
    assert torch.equal(o[fine], clean[0][fine]) and torch.equal(lse, clean[1])
    got, want = o.double().cpu()[~fine.cpu()], ref_o[~fine.cpu()]
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize(("group", "nodes"), [(1, 1), (4, 8), (8, 8), (8, 16), (8, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights_beside_a_large_one(group: int, nodes: int, dtype: torch.dtype) -> None:
    """4000 keys at 2^-25.5 of the one that dominates, whose own value is 0: they are the output.  So many sequences that
    few items are cut.  In float16 a weight is rounded to a multiple of 2^-31 of the largest at worst."""
    count, dim, batch = 4000, 64, 160
    p = problem(1, group, 1, nodes, dim, count + 1, [count + 1], dtype, seed=nodes, tree=False)
    for name in ("q", "k_cache", "k_tree", "v_tree"):
        p[name].zero_()
    p["q"][..., 0] = 1.0
    p["k_cache"][..., 0] = -25.5 * math.log(2.0)
    p["k_tree"][..., 0] = -60.0
    p["v_cache"] = ((p["v_cache"].float().abs() + 0.5) * 64.0).to(dtype)
    p["k_cache"][:, :, 0] = 0.0
    p["v_cache"][:, :, 0] = 0.0
    many = {n: None if t is None else t.cuda().repeat(batch, *[1] * (t.ndim - 1)) for n, t in p.items()}
    o, lse = tree_attention(**many, scale=1.0, return_lse=True)
    ref_o, ref_lse, spread = tree_attention_reference(**p, scale=1.0)
    largest = float(p["v_cache"].abs().max())
    bound = (2.0 * ROUND[dtype] + 2.0**-12) * spread + (count * 2.0**-32 * largest if dtype == torch.float16 else 0.0)
    err = (o.double().cpu() - ref_o).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert torch.allclose(lse.double().cpu(), ref_lse.expand(batch, -1, -1), atol=2e-4)
    check_device_status()


@pytest.mark.parametrize("place", [1, 4, 7, 10, 2, 11])
def test_library_refuses_strides_of_zero(place: int) -> None:
    """Rows or heads that are one in memory: no tensor map describes them."""
    strides = [64] * 12
    strides[place] = 0
    args = {"q": 0x1000, "k": 0x1000, "v": 0x1000, "k_tree": 0x1000, "v_tree": 0x1000, "strides": (ctypes.c_int64 * 12)(*strides),
            "kv_lens": 0x1000, "parents": None, "parent_stride": 0, "tree_sizes": None, "o": 0x1000, "lse": None, "workspace": None,
            "workspace_bytes": 0, "batch": 1, "q_heads": 4, "kv_heads": 2, "nodes": 3, "seq_kv": 16, "head_dim": 64, "dtype": 1,
            "scale": 0.125, "stream": None}
    assert _native.load().tk_tree_attn(*args.values()) == 1


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("across", [(0,), (1,), (2,), (0, 1), (0, 1, 2)])
def test_trees_that_repeat_in_memory(across: tuple[int, ...]) -> None:
    g = on_gpu(problem(3, 8, 4, 5, 64, 70, [70, 1, 40], torch.bfloat16, seed=13))
    one = {}
    for name in ("k_tree", "v_tree"):
        part = g[name]
        for axis in across:
            part = part.narrow(axis, 0, 1)
        one[name] = part.expand(3, 4, 5, 64)
    ref = tree_attention(**{**g, **{n: t.contiguous() for n, t in one.items()}})
    assert torch.equal(tree_attention(**{**g, **one}), ref)
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("which", ["q", "k_cache", "v_cache", "k_tree", "v_tree"])
def test_a_gradient_through_it_is_an_error(which: str) -> None:
    """No derivative: a loss that depends on it says so in its backward pass, it does not lose a term."""
    g = on_gpu(problem(2, 4, 2, 5, 64, 40, [40, 7], torch.bfloat16, seed=14))
    ref, ref_lse = tree_attention(**g, return_lse=True)
    g[which].requires_grad_(True)
    o, lse = tree_attention(**g, return_lse=True)
    assert torch.equal(o, ref) and torch.equal(lse, ref_lse)
    for out in (o, lse, tree_attention(**g)):
        with pytest.raises(RuntimeError, match="no derivative"):
            out.float().sum().backward()
    assert g[which].grad is None
    with torch.no_grad():
        o = tree_attention(**g)
    assert not o.requires_grad and torch.equal(o, ref)
    o = tree_attention(**{**g, which: g[which].detach()})
    assert not o.requires_grad and torch.equal(o, ref)
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("which", ["q", "v_cache", "k_tree"])
def test_a_tangent_through_it_is_an_error(which: str) -> None:
    g = on_gpu(problem(2, 4, 2, 5, 64, 40, [40, 7], torch.bfloat16, seed=14))
    with torch.autograd.forward_ad.dual_level():
        g[which] = torch.autograd.forward_ad.make_dual(g[which], torch.ones_like(g[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            tree_attention(**g)
