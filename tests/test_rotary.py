"""``tklab.kernels.rotary``: tables (CPU), refusals (CPU) and the kernel against the 64-bit reference (GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle.speculative_oracle import rotary_reference
from tklab import _native
from tklab.kernels.flash_attention import check_device_status
from tklab.kernels.rope_attention import rope_tables, torch_rope
from tklab.kernels.rotary import rotary, rotary_tables

gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU is required")

# Unit roundoff of the output type, and the smallest subnormal step's half.
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = 2.0**-25


def assert_rotated(y: torch.Tensor, x: torch.Tensor, ref: torch.Tensor, gain: float = 1.0) -> None:
    """One rounding of the result, plus three fp32 roundings of terms no larger than the pair's inputs."""
    size = gain * 2.0 * x.double().abs().amax(-1, keepdim=True)
    bound = ROUND[y.dtype] * ref.abs() + 3.0 * 2.0**-24 * size * (1.0 + ROUND[y.dtype]) + TINY
    assert bool(((y.double() - ref).abs() <= bound).all())


# ------------------------------------------------------------------ tables
def test_plain_tables_equal_the_rope_attention_tables() -> None:
    for mine, theirs in zip(rotary_tables(50, 64), rope_tables(50, 64), strict=True):
        assert torch.equal(mine, theirs)


def test_scaled_tables() -> None:
    n, r, f, orig = 64, 32, 4.0, 1024
    index = torch.arange(r // 2, dtype=torch.float64)
    rates = 10000.0 ** (-2.0 * index / r)

    def rates_of(**kwargs: object) -> torch.Tensor:
        cos, sin = rotary_tables(2, r, factor=f, **kwargs)
        return torch.atan2(sin[1].double(), cos[1].double())

    assert torch.allclose(rates_of(scaling="linear"), rates / f, rtol=1e-5)
    ntk = rates_of(scaling="ntk")
    assert ntk[0] == pytest.approx(1.0, rel=1e-6) and ntk[-1] == pytest.approx(float(rates[-1]) / f, rel=1e-4)
    turns = orig * rates / (2.0 * math.pi)
    bands = rates_of(scaling="bands", original_positions=orig)
    assert torch.allclose(bands[turns >= 4.0], rates[turns >= 4.0], rtol=1e-5)
    assert torch.allclose(bands[turns <= 1.0], rates[turns <= 1.0] / f, rtol=1e-5)
    between = (turns > 1.0) & (turns < 4.0)
    assert bool(between.any()) and bool((bands[between] < rates[between]).all() and (bands[between] > rates[between] / f).all())
    yarn = rates_of(scaling="yarn", original_positions=orig)
    assert torch.allclose(yarn[turns > 40.0], rates[turns > 40.0], rtol=1e-5)
    assert torch.allclose(yarn[turns < 0.5], rates[turns < 0.5] / f, rtol=1e-5)
    cos, sin = rotary_tables(n, r, scaling="yarn", factor=f, original_positions=orig)
    assert torch.allclose(cos.square() + sin.square(), torch.tensor((0.1 * math.log(f) + 1.0) ** 2), rtol=1e-5)
    for scaling in ("linear", "ntk", "yarn", "bands"):  # factor 1 changes nothing
        for a, b in zip(rotary_tables(n, r, scaling=scaling, original_positions=orig), rotary_tables(n, r), strict=True):
            assert torch.allclose(a, b, atol=1e-6)


@pytest.mark.parametrize(
    ("kwargs", "match"),
    [
        ({"n_positions": 0}, "at least one"),
        ({"rotary_dim": 7}, "even"),
        ({"scaling": "other"}, "scaling must be"),
        ({"factor": 0.5}, "factor"),
        ({"scaling": "yarn", "factor": 2.0}, "original_positions"),
    ],
)
def test_tables_refuse(kwargs: dict, match: str) -> None:
    with pytest.raises(ValueError, match=match):
        rotary_tables(**{"n_positions": 8, "rotary_dim": 16, **kwargs})


# ---------------------------------------------------------------- refusals
def test_rotary_refuses() -> None:
    q = torch.zeros(2, 4, 6, 32, dtype=torch.bfloat16)
    cos, sin = rotary_tables(6, 32)
    for args, kwargs, match in [
        ((q[0], q, cos, sin), {}, "shaped"),
        ((q, q[:, :, :5], cos, sin), {}, "agree"),
        ((q.float(), q.float(), cos, sin), {}, "dtype"),
        ((q, q.half(), cos, sin), {}, "dtype"),
        ((q[..., :30], q[..., :30], cos[:, :8], sin[:, :8]), {}, "multiple of 8"),
        ((q[:0], q[:0], cos, sin), {}, "empty"),
        ((q, q, cos, sin[:4]), {}, "one shape"),
        ((q, q, *rotary_tables(6, 64)), {}, "wider"),
        ((q, q, cos.int(), sin.int()), {}, "floating"),
        ((q, q, cos, sin), {"layout": "other"}, "layout"),
        ((q, q, cos, sin), {}, "CUDA"),
    ]:
        with pytest.raises(ValueError, match=match):
            rotary(*args, **kwargs)


@pytest.mark.parametrize(
    ("kwargs", "status"),
    [
        ({"q": None}, 1), ({"cos": None}, 1), ({"k": None}, 1), ({"batch": 0}, 1), ({"q_heads": 0}, 1),
        ({"table_rows": 0}, 1), ({"table_rows": 3}, 1), ({"head_dim": 20}, 2), ({"head_dim": 264}, 2),
        ({"rotary_dim": 15}, 2), ({"rotary_dim": 66}, 2), ({"dtype": 4}, 2), ({"q": 0x1008}, 3),
        ({"positions": 0x2002}, 3), ({"strides": (64, 68, 64)}, 3),
    ],
)
def test_library_refuses_before_launch(kwargs: dict, status: int) -> None:
    import ctypes

    args = {"q": 0x1000, "k": 0x1000, "q_out": 0x1000, "k_out": 0x1000, "cos": 0x1000, "sin": 0x1000,
            "positions": None, "positions_64": 0, "batch": 1, "q_heads": 2, "kv_heads": 1, "seq": 4, "head_dim": 64,
            "rotary_dim": 64, "table_rows": 4, "q_strides": (512, 256, 64), "k_strides": (256, 256, 64), "dtype": 1,
            "interleaved": 0, "transpose": 0, "stream": None}
    strides = kwargs.pop("strides", args["q_strides"])
    args.update(kwargs)
    args["q_strides"] = (ctypes.c_int64 * 3)(*strides)
    args["k_strides"] = (ctypes.c_int64 * 3)(*args["k_strides"])
    assert _native.load().tk_rotary(*args.values()) == status


# --------------------------------------------------------------------- GPU
def make(shape, dtype, gen, order="bhsd"):
    b, h, s, d = shape
    if order == "bshd":
        return torch.randn(b, s, h, d, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize(
    ("dim", "rotary_dim"),
    [(64, 64), (128, 128), (128, 64), (96, 24), (80, 20), (80, 40), (72, 72), (8, 8), (8, 2), (40, 6), (256, 256), (128, 30)],
)
@pytest.mark.parametrize("order", ["bhsd", "bshd"])
def test_rotary_matches_reference(dtype: torch.dtype, layout: str, dim: int, rotary_dim: int, order: str) -> None:
    gen = torch.Generator(device="cuda").manual_seed(dim + rotary_dim)
    q, k = make((2, 6, 7, dim), dtype, gen, order), make((2, 3, 7, dim), dtype, gen, order)
    cos, sin = rotary_tables(7, rotary_dim, device="cuda")
    for x, y in zip((q, k), rotary(q, k, cos, sin, layout=layout), strict=True):
        assert y.is_contiguous() and y.shape == x.shape and y.dtype == dtype
        assert_rotated(y.cpu(), x.cpu(), rotary_reference(x.cpu(), cos.cpu(), sin.cpu(), layout=layout))
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("seq", [1, 2, 33, 300])
@pytest.mark.parametrize("wide", [False, True])
def test_positions(seq: int, wide: bool) -> None:
    gen = torch.Generator(device="cuda").manual_seed(seq)
    q, k = make((3, 4, seq, 64), torch.bfloat16, gen, "bshd"), make((3, 1, seq, 64), torch.bfloat16, gen)
    cos, sin = rotary_tables(1000, 64, scaling="yarn", factor=8.0, original_positions=256, device="cuda")
    positions = torch.randint(0, 1000, (3, seq), generator=gen, device="cuda", dtype=torch.int64 if wide else torch.int32)
    for x, y in zip((q, k), rotary(q, k, cos, sin, positions=positions), strict=True):
        assert_rotated(y.cpu(), x.cpu(), rotary_reference(x.cpu(), cos.cpu(), sin.cpu(), positions=positions.cpu()), gain=1.21)
    shared = rotary(q, None, cos, sin, positions=positions[0])[0]
    assert torch.equal(shared, rotary(q, None, cos, sin, positions=positions[:1].expand(3, seq))[0])
    check_device_status()


@pytest.mark.gpu
@gpu
def test_position_outside_the_tables_is_reported_and_kept() -> None:
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = make((1, 2, 4, 64), torch.float16, gen)
    cos, sin = rotary_tables(8, 64, device="cuda")
    positions = torch.tensor([[3, -1, 8, 2**30]], device="cuda")
    y, none = rotary(q, None, cos, sin, positions=positions)
    assert none is None
    with pytest.raises(RuntimeError, match="invalid argument"):
        check_device_status()
    assert torch.equal(y[:, :, 1:], q[:, :, 1:])
    assert_rotated(y.cpu(), q.cpu(), rotary_reference(q.cpu(), cos.cpu(), sin.cpu(), positions=positions.cpu()))
    check_device_status()


@pytest.mark.gpu
@gpu
def test_odd_strides_and_alignment() -> None:
    gen = torch.Generator(device="cuda").manual_seed(6)
    cos, sin = rotary_tables(9, 32, device="cuda")
    big = torch.randn(2, 9, 5, 47, generator=gen, device="cuda").to(torch.bfloat16)
    odd = big[..., 3:35].transpose(1, 2)  # rows at an odd stride, off any 16-byte boundary
    padded = torch.randn(2, 5, 9, 48, generator=gen, device="cuda").to(torch.bfloat16)[..., 16:48]
    columns = torch.randn(2, 5, 32, 9, generator=gen, device="cuda").to(torch.bfloat16).transpose(2, 3)
    broadcast = torch.randn(2, 1, 9, 32, generator=gen, device="cuda").to(torch.bfloat16).expand(2, 5, 9, 32)
    for x in (odd, padded, columns, broadcast):
        y, z = rotary(x, x[:, :2], cos.double(), sin.double())
        assert_rotated(y.cpu(), x.cpu(), rotary_reference(x.cpu(), cos.cpu(), sin.cpu()))
        assert torch.equal(z, y[:, :2])
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize(("dim", "rotary_dim"), [(64, 64), (96, 24), (80, 20)])
def test_gradient(layout: str, dim: int, rotary_dim: int) -> None:
    """Against the transposed rotation in 64 bits, and <dy, R(x + e) - R(x)> against <grad, e> by differences."""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = make((2, 6, 9, dim), torch.float16, gen, "bshd").requires_grad_(True)
    k = make((2, 2, 9, dim), torch.float16, gen).requires_grad_(True)
    cos, sin = rotary_tables(40, rotary_dim, scaling="yarn", factor=4.0, original_positions=16, device="cuda")
    positions = torch.randint(0, 40, (2, 9), generator=gen, device="cuda")
    dq, dk = make((2, 6, 9, dim), torch.float16, gen), make((2, 2, 9, dim), torch.float16, gen, "bshd")
    out = rotary(q, k, cos, sin, positions=positions, layout=layout)
    grads = torch.autograd.grad(out, (q, k), (dq, dk))
    host = {"positions": positions.cpu(), "layout": layout}
    for g, d, x in zip(grads, (dq, dk), (q, k), strict=True):
        assert g.shape == x.shape
        assert_rotated(g.cpu(), d.cpu(), rotary_reference(d.cpu(), cos.cpu(), sin.cpu(), transpose=True, **host), gain=1.14)
        e = torch.randn(x.shape, generator=gen, device="cuda").cpu().double()
        xc = x.detach().cpu().double()
        moved = rotary_reference(xc + e, cos.cpu(), sin.cpu(), **host) - rotary_reference(xc, cos.cpu(), sin.cpu(), **host)
        left, right = (d.cpu().double() * moved).sum(), (g.cpu().double() * e).sum()
        # Every gradient entry is off by at most a rounding and a bit.
        assert abs(float(left - right)) <= float((g.cpu().double() * e).abs().sum()) * 2.0**-10
    # One output used alone, and a broadcast input.
    assert torch.equal(torch.autograd.grad(rotary(q, k, cos, sin, positions=positions, layout=layout)[1], k, dk)[0], grads[1])
    one = torch.zeros(2, 1, 9, dim, dtype=torch.float16, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(rotary(one.expand(2, 6, 9, dim), None, cos, sin, positions=positions, layout=layout)[0], one, dq)
    assert torch.allclose(g.float(), grads[0].float().sum(1, keepdim=True), atol=6 * 2.0**-10 * 8)
    check_device_status()


@pytest.mark.gpu
@gpu
def test_agrees_with_torch_rope_and_other_streams() -> None:
    gen = torch.Generator(device="cuda").manual_seed(11)
    q = make((2, 3, 130, 128), torch.bfloat16, gen)
    cos, sin = rotary_tables(130, 128, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y, _ = rotary(q, None, cos, sin)
    side.synchronize()
    assert_rotated(y.cpu(), q.cpu(), torch_rope(q.double(), cos.double(), sin.double()).cpu())
    check_device_status()


@pytest.mark.gpu
@gpu
def test_gradient_of_the_gradient_and_without_positions() -> None:
    """The rotation is linear: its second derivative is the rotation of the cotangent's cotangent."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    cos, sin = rotary_tables(5, 64, device="cuda")
    q = make((1, 2, 5, 64), torch.float16, gen).requires_grad_(True)
    k = make((1, 1, 5, 64), torch.float16, gen).requires_grad_(True)
    dq, dk = (make(x.shape, torch.float16, gen).requires_grad_(True) for x in (q, k))
    gq, gk = torch.autograd.grad(rotary(q, k, cos, sin), (q, k), (dq, dk), create_graph=True)
    v, w = make(q.shape, torch.float16, gen), make(k.shape, torch.float16, gen)
    for got, x in zip(torch.autograd.grad((gq, gk), (dq, dk), (v, w)), (v, w), strict=True):
        assert_rotated(got.cpu(), x.cpu(), rotary_reference(x.cpu(), cos.cpu(), sin.cpu()))
    (g,) = torch.autograd.grad(rotary(q, k.detach(), cos, sin)[0], q, dq.detach())
    assert torch.equal(g, gq)
    check_device_status()


@pytest.mark.gpu
@gpu
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("order", ["bhsd", "bshd"])
def test_a_tangent_through_it_is_an_error(which: int, order: str) -> None:
    """Forward-mode differentiation is refused, with requires_grad or without; a tangent is not lost."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = rotary_tables(5, 64, device="cuda")
    x = [make((1, 2, 5, 64), torch.float16, gen, order) for _ in range(2)]
    with torch.autograd.forward_ad.dual_level():
        x[which] = torch.autograd.forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            rotary(*x, cos, sin)
        x[which].requires_grad_(True)
        with pytest.raises(RuntimeError):
            rotary(*x, cos, sin)
