"""Rotary positions of several axes (row and column of an image, time as well in a video).

The reference has no such operator; names, checks and errors follow
:mod:`deformops_b200.registry.msda`.
"""

from __future__ import annotations

import functools
import struct
from typing import Sequence

import torch
from torch import Tensor

from .. import attention_ops as _ops  # noqa: F401  (defines the operators)
from .._loader import load_library
from ..core.errors import NoBackendError
from ..core.runtime import sm_version_for
from ..core.sanitize import check_rotary_call
from .msda import Backend, _native_path, msda

__all__ = ["rotary"]

_MAX_PAIRS = 128


class _Plan:
    """Frequency and axis of every pair, as lists and as the native path's packed doubles and ints."""

    def __init__(self, sections: tuple[int, ...], base: float, joint: bool):
        if not base > 0.0:
            raise ValueError(f"base must be positive, got {base}")
        if any(n < 0 for n in sections):
            raise ValueError(f"sections {sections} are pairs of channels per axis: none may be negative")
        total = sum(sections)
        self.frequencies: list[float] = []
        self.axes: list[int] = []
        for axis, count in enumerate(sections):
            first = len(self.axes)
            for i in range(count):
                self.frequencies.append(base ** (-(first + i) / total if joint else -i / count))
                self.axes.append(axis)
        self.packed = struct.pack(f"{total}d{total}i", *self.frequencies, *self.axes)


@functools.lru_cache(maxsize=256)
def _plan(sections: tuple[int, ...], base: float, joint: bool) -> _Plan:
    return _Plan(sections, base, joint)


@functools.lru_cache(maxsize=256)
def _even_sections(head_dim: int, axes: int) -> tuple[int, ...]:
    if axes == 0 or head_dim % (2 * axes) != 0:
        raise ValueError(f"a head of {head_dim} channels has no equal number of pairs for {axes} axes: pass sections")
    return (head_dim // (2 * axes),) * axes


def rotary(x: Tensor, positions: Tensor, *, sections: Sequence[int] | None = None, base: float = 10000.0,
           interleaved: bool = False, joint: bool = False, backend: Backend | None = None) -> Tensor:
    """``x (B,N,G,D)`` with its pairs of channels turned by ``positions (B,N,A)`` or ``(N,A)``.

    ``sections`` says how many pairs turn with each of the ``A`` axes, in order (default: ``D / 2``
    shared out evenly); channels behind them pass through.  Pair ``i`` of an axis with ``n`` pairs turns
    by ``position * base ** (-i / n)``; with ``joint`` there is one series over all pairs,
    ``base ** (-j / sum(sections))``, whatever their axis.  Pairs are the channels ``(i, i + P)`` of the
    ``2 P`` that turn, or with ``interleaved`` the neighbours ``(2 i, 2 i + 1)``.

    Positions are float32, float64, int32 or int64, of any size and sign (angles are formed in 64
    bits; those of float32 positions to 2^-28 of a turn up to 2^20 turns), and take no gradient.  The result is dense and has the type of ``x`` (float32, float16, bfloat16).
    """
    heads_dim = x.shape[3] if x.dim() == 4 else 0
    if sections is None:
        sections = _even_sections(heads_dim, positions.shape[-1]) if heads_dim else ()
    elif type(sections) is not tuple:
        sections = tuple(int(n) for n in sections)
    if backend is None or backend is Backend.CUDA:
        native = _native_path(x)
        if native is not None:
            out = native.rotary(x, positions, _plan(sections, base, joint).packed, len(sections), interleaved)
            if out is not None:
                return out
    msda._only_cuda(backend)
    check_rotary_call(x, positions, sections)
    reason = None
    if x.device.type != "cuda":
        reason = f"tensors are on {x.device}; the kernels need a CUDA device (no CPU path)"
    elif sm_version_for(x.device)[0] != 10:
        reason = "the kernels are built for sm_100a only"
    elif x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        reason = f"dtype {x.dtype} is not float32, float16 or bfloat16"
    elif sum(sections) > _MAX_PAIRS or len(sections) > 255:
        reason = f"{sum(sections)} pairs; at most {_MAX_PAIRS} are turned"
    if reason is not None:
        raise NoBackendError(f"rotary cannot run this call: {reason}")
    plan = _plan(sections, base, joint)
    load_library()
    return torch.ops.deformops_b200.rotary_turn(x, positions, plan.frequencies, plan.axes, bool(interleaved), False)
