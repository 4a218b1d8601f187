"""Rotary positions on queries and keys (B200): any positions, both layouts,
part of the head, long-context tables, forward and backward.

:func:`rotary` rotates ``q`` (batch, q_heads, seq, head_dim) and ``k``
(batch, kv_heads, seq, head_dim) in one launch (``tk_rotary``).  With ``r``
the width of the tables times two, pair ``i`` of a row at position ``p`` is

* ``layout="half"``: columns ``(i, i + r/2)``,
* ``layout="interleaved"``: columns ``(2i, 2i + 1)``,

and in fp32, rounded once to the input dtype, ``y1 = x1 cos[p][i] - x2
sin[p][i]``, ``y2 = x2 cos[p][i] + x1 sin[p][i]``; columns from ``r`` on are
copied.  The arithmetic is that of the reference's rotate-half ``rope``
(``src/tklab/kernels/rope.py:27-74``); :func:`tklab.kernels.rope_attention
.attention_rope` fuses that one form (whole heads of 64 or 128, positions
0..S-1) into the attention forward, this operator serves the rest: decode
steps and drafted tokens at their own positions, partial heads, interleaved
pairs, projections in (batch, seq, heads, dim) order (any strides whose rows
are contiguous are read in place; the results are contiguous (batch, heads,
seq, head_dim), as the attention kernels take them).

:func:`rotary_tables` makes the tables in fp64, optionally scaled for long
contexts.  The tables are constants: no gradient flows to them.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from tklab import _native
from tklab.kernels._plans import Plans, _after_launch, _stream, at_device, dense, meta, row_strides, stride_array
from tklab.kernels.flash_attention import _NATIVE_DTYPE

ROTARY_LAYOUTS = ("half", "interleaved")
ROTARY_SCALINGS = ("none", "linear", "ntk", "yarn", "bands")
MAX_ROTARY_HEAD_DIM = 256


def rotary_tables(
    n_positions: int,
    rotary_dim: int,
    *,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original_positions: int | None = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    low_band: float = 1.0,
    high_band: float = 4.0,
    device: torch.device | str = "cpu",
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosine and sine tables (n_positions, rotary_dim // 2), fp32 from fp64 angles ``p * w_i``.

    ``w_i = base ** (-2 i / rotary_dim)``, changed by ``scaling`` to stretch a
    context of ``original_positions`` by ``factor``:

    * ``"linear"``: ``w_i / factor`` (positions interpolated);
    * ``"ntk"``: the base raised to ``base * factor ** (r / (r - 2))``, which
      keeps the fastest pair and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times over the
      original context are kept, those below ``beta_slow`` divided by
      ``factor``, a linear ramp over the pair index between; both tables are
      multiplied by ``0.1 ln(factor) + 1``;
    * ``"bands"``: pairs with at least ``high_band`` turns over the original
      context are kept, those with at most ``low_band`` divided by
      ``factor``, and between them the two are mixed linearly in the turns.
    """
    if n_positions <= 0:
        raise ValueError("rotary tables need at least one position")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be an even number from 2")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"rotary scaling must be one of {ROTARY_SCALINGS}")
    if not (base > 1.0 and factor >= 1.0):
        raise ValueError("rotary tables need base > 1 and factor >= 1")
    if scaling in ("yarn", "bands") and not original_positions:
        raise ValueError(f"rotary scaling {scaling!r} needs original_positions")
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else base
    index = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    rates = base ** (-2.0 * index / rotary_dim)
    gain = 1.0
    if scaling == "linear":
        rates = rates / factor
    elif scaling == "yarn":

        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        rates = rates * (1.0 - ramp) + rates / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling == "bands":
        turns = original_positions * rates / (2.0 * math.pi)
        keep = ((turns - low_band) / (high_band - low_band)).clamp(0.0, 1.0)
        rates = rates * keep + rates / factor * (1.0 - keep)
    angles = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * rates
    return (gain * angles.cos()).to(torch.float32), (gain * angles.sin()).to(torch.float32)


_PLANS = Plans()


def _plan(
    q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
    positions: torch.Tensor | None, layout: str,
) -> tuple:
    """Check the contract; return what a call with this metadata passes to the library.

    The first entry says whether every tensor can be read in place.
    """
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"rotary layout must be one of {ROTARY_LAYOUTS}")
    if q.ndim != 4:
        raise ValueError("rotary expects q shaped (batch, heads, sequence, dim)")
    batch, q_heads, seq, head_dim = q.shape
    if k is not None and (k.ndim != 4 or k.shape[0] != batch or k.shape[2] != seq or k.shape[3] != head_dim):
        raise ValueError("q and k must agree on batch, sequence and head_dim")
    if 0 in q.shape or (k is not None and 0 in k.shape):
        raise ValueError("rotary does not support empty dimensions")
    if q.dtype not in _NATIVE_DTYPE or (k is not None and k.dtype != q.dtype):
        raise ValueError("q and k must share one dtype: float16 or bfloat16")
    if head_dim % 8 or head_dim > MAX_ROTARY_HEAD_DIM:
        raise ValueError(f"rotary requires head_dim to be a multiple of 8 up to {MAX_ROTARY_HEAD_DIM}")
    if cos.ndim != 2 or cos.shape != sin.shape or 0 in cos.shape:
        raise ValueError("cos and sin must be (positions, rotary_dim // 2) tables of one shape")
    if 2 * cos.shape[1] > head_dim:
        raise ValueError("the tables are wider than half of head_dim")
    if not (cos.is_floating_point() and sin.is_floating_point()):
        raise ValueError("cos and sin must be floating-point tables")
    device = q.device
    if device.type != "cuda":
        raise ValueError("rotary requires CUDA tensors")
    if cos.device != device or sin.device != device or (k is not None and k.device != device):
        raise ValueError("q, k, cos, and sin must be on the same device")
    if positions is None:
        if cos.shape[0] < seq:
            raise ValueError("the tables have fewer rows than the sequence")
    else:
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != device:
            raise ValueError("positions must be an int32 or int64 tensor on q's device")
        if positions.shape not in ((batch, seq), (seq,)):
            raise ValueError("positions must be shaped (batch, sequence) or (sequence,)")
    q_strides = row_strides(q)
    k_strides = (0, 0, 0) if k is None else row_strides(k)
    in_place = (
        q_strides is not None and k_strides is not None
        and all(t.dtype == torch.float32 and t.is_contiguous() for t in (cos, sin))
        and (positions is None or (positions.ndim == 2 and positions.is_contiguous()))
    )
    return (
        in_place, q.get_device(), (batch, 0 if k is None else k.shape[1], seq, head_dim),
        stride_array(*(q_strides or ())), stride_array(*(k_strides or ())),
        0 if positions is None else int(positions.dtype == torch.int64),
        batch, q_heads, 0 if k is None else k.shape[1], seq, head_dim, 2 * cos.shape[1], cos.shape[0],
        _NATIVE_DTYPE[q.dtype], int(layout == "interleaved"),
    )


def _table(t: torch.Tensor) -> torch.Tensor:
    t = t.detach()
    return t.to(torch.float32, copy=bool(t.data_ptr() & 15), memory_format=torch.contiguous_format).contiguous()


def _launch(
    q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
    positions: torch.Tensor | None, layout: str, transpose: int,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Check (or recall) and make the library call, into fresh contiguous outputs."""
    key = (
        q.shape, q.stride(), q.dtype, q.get_device(), meta(k), cos.shape, cos.stride(), cos.dtype, cos.get_device(),
        sin.shape, sin.stride(), sin.dtype, sin.get_device(), meta(positions), layout,
    )
    plan = _PLANS.get(key) or _PLANS.keep(key, _plan(q, k, cos, sin, positions, layout))
    (in_place, device, k_shape, q_strides, k_strides, wide, batch, q_heads, kv_heads, seq, head_dim, rotary_dim, rows,
     dtype, interleaved) = plan
    q_ptr, k_ptr = q.data_ptr(), 0 if k is None else k.data_ptr()
    cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    if not in_place or (q_ptr | k_ptr | cos_ptr | sin_ptr) & 15:
        if positions is not None:
            positions = positions.expand(batch, seq).contiguous()
        return _launch(
            dense(q), None if k is None else dense(k), _table(cos), _table(sin), positions, layout, transpose
        )
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    with at_device(device):
        status = _native.load().tk_rotary(
            q_ptr, k_ptr, q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(), cos_ptr, sin_ptr,
            0 if positions is None else positions.data_ptr(), wide, batch, q_heads, kv_heads, seq, head_dim,
            rotary_dim, rows, q_strides, k_strides, dtype, interleaved, transpose, _stream(q),
        )
    _native.check(status, "tk_rotary")
    _after_launch(q.device)
    return q_out, k_out


class _RotaryFunction(torch.autograd.Function):
    """Autograd bridge: the backward is the transposed rotation of both gradients in one launch."""

    @staticmethod
    def forward(ctx: Any, q, k, cos, sin, positions, layout):
        """Rotate and keep the tables and positions."""
        ctx.save_for_backward(cos, sin, positions)
        ctx.layout = layout
        ctx.set_materialize_grads(False)
        return _launch(q, k, cos, sin, positions, layout, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dq, dk):
        """Input gradients of whichever outputs were used."""
        cos, sin, positions = ctx.saved_tensors
        gq = gk = None
        if dq is not None:
            gq, gk = _launch(dq, dk, cos, sin, positions, ctx.layout, 1)
        elif dk is not None:
            gk, _ = _launch(dk, None, cos, sin, positions, ctx.layout, 1)
        return gq, gk, None, None, None, None


def rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    layout: str = "half",
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate ``q`` and ``k`` (or ``q`` alone, ``k=None``) by the tables' rows ``positions``.

    ``positions``: (batch, seq) or (seq,) int32/int64, 0..seq-1 when None.  A
    position outside the tables leaves its rows as they are and is reported
    by :func:`tklab.kernels.flash_attention.check_device_status`.  Returns
    contiguous (batch, heads, seq, head_dim) tensors; differentiable in ``q``
    and ``k``.
    """
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RotaryFunction.apply(q, k, cos, sin, positions, layout)
    return _launch(q, k, cos, sin, positions, layout, 0)
