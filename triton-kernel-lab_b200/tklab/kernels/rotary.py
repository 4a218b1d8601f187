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

import torch

from tklab._tensors import binding, dense
from tklab.kernels.flash_attention import _NATIVE_DTYPE, _after_launch

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


def _prepare(
    q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None
) -> tuple:
    """Check the contract; return the arguments with whatever the kernel cannot read in place copied."""
    if q.ndim != 4:
        raise ValueError("rotary expects q shaped (batch, heads, sequence, dim)")
    batch, _, seq, head_dim = q.shape
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
        positions = positions.expand(batch, seq).contiguous()

    def table(t: torch.Tensor) -> torch.Tensor:
        t = t.detach().to(torch.float32).contiguous()
        return t.clone() if t.data_ptr() % 16 else t

    return dense(q), None if k is None else dense(k), table(cos), table(sin), positions


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
    and ``k`` (backward passes of any order; forward mode is refused).
    """
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"rotary layout must be one of {ROTARY_LAYOUTS}")
    interleaved = layout == "interleaved"
    out = binding.rotary(q, k, cos, sin, positions, interleaved)
    if out is None:
        out = binding.rotary(*_prepare(q, k, cos, sin, positions), interleaved)
        if out is None:
            raise ValueError("rotary: unsupported arguments")
    _after_launch(q.device)
    return out
