"""Checked calls, remembered by their tensors' metadata.

Checking a call's shapes, strides, dtypes and devices costs more host time
than launching it.  The serving operators (``rotary``, ``tree_attention``,
``verify_draft``, ``commit_draft``) are called with the same ones step after
step, so each keeps what its checks derived, keyed by that metadata alone:
no address, value or tensor is kept, and pointers (alignment included) are
looked at in every call.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from tklab.kernels.flash_attention import _after_launch, _on_device, _stream

MAX_PLANS = 1024


class Plans(dict):
    """Plans by metadata; emptied when it has grown past ``MAX_PLANS`` entries."""

    def keep(self, key: tuple, plan: tuple) -> tuple:
        """Remember ``plan``."""
        if len(self) >= MAX_PLANS:
            self.clear()
        self[key] = plan
        return plan


def meta(x: torch.Tensor | None) -> tuple | None:
    """What a plan may depend on in ``x``."""
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


@functools.lru_cache(maxsize=1024)
def stride_array(*strides: int) -> ctypes.Array:
    """Strides as the C array that the library reads (never written)."""
    return (ctypes.c_int64 * len(strides))(*strides)


def row_strides(x: torch.Tensor) -> tuple[int, ...] | None:
    """Strides of every dimension but the last (0 for dimensions of size 1), or None if
    the kernels cannot read rows in place: contiguous, at strides that are multiples of 8."""
    *outer, last = x.stride()
    if last != 1 and x.shape[-1] > 1:
        return None
    strides = tuple(0 if n == 1 else s for n, s in zip(x.shape, outer))
    return None if any(s % 8 for s in strides) else strides


def dense(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if its rows can be read in place at a 16-byte aligned address, else a contiguous copy."""
    if row_strides(x) is None or x.data_ptr() & 15:
        return x.clone(memory_format=torch.contiguous_format)
    return x


class at_device(_on_device):
    """:class:`_on_device` for a device index."""

    __slots__ = ()

    def __init__(self, index: int) -> None:
        self._ctx = None if index == torch.cuda.current_device() else torch.cuda.device(index)


__all__ = ["Plans", "_after_launch", "_stream", "at_device", "dense", "meta", "row_strides", "stride_array"]
