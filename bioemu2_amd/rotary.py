"""Rotary positions on MI355X, trainable.

``RelativePosition`` and the bias of ``attention`` learn a value for each bucket
of distance; ``rotary`` puts positions into q and k instead, by turning pairs of
their values, so that scores depend on distances alone, at any length and with
nothing to learn.  ``rotary_frequencies`` lays out the frequencies, also for
contexts longer than those trained on.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch import Tensor

from . import _ops
from ._lib import torch_op
from .relative_position import _int32

SCALINGS = ("linear", "base", "parts")


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       length: int | None = None, turns: tuple[float, float] = (1.0, 32.0), device=None) -> Tensor:
    """Radians a position (64 bits, [dim / 2]) of the pairs of ``dim`` values: ``base ** (-2 i / dim)``.

    For contexts ``factor`` times as long, ``scaling`` slows them:
    "linear": all by ``factor``;
    "base": by a longer base, ``base * factor ** (dim / (dim - 2))``: the slowest by ``factor``, the fastest not;
    "parts": by how often a pair turns over the ``length`` trained on: those below ``turns[0]`` by ``factor``, those
    above ``turns[1]`` not, between them a linear share of both (``rotary``'s magnitude is then usually
    ``0.1 ln(factor) + 1``)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if not base > 0 or not factor > 0:
        raise ValueError(f"rotary_frequencies: base {base}, factor {factor}")
    if scaling is not None and scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling {scaling!r}, one of {SCALINGS}")
    if scaling is None and factor != 1.0:
        raise ValueError("rotary_frequencies: a factor comes with its scaling")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "parts":
        if length is None or length < 1 or not turns[1] > turns[0]:
            raise ValueError(f"rotary_frequencies: scaling 'parts' takes a length and growing turns, got {length}, {turns}")
        kept = [min(max((length * x / (2 * math.pi) - turns[0]) / (turns[1] - turns[0]), 0.0), 1.0) for x in f]
        f = [x * (k + (1.0 - k) / factor) for x, k in zip(f, kept)]
    return torch.tensor(f, dtype=torch.float64, device=device)


def rotary(q: Tensor | None, k: Tensor | None, positions: Tensor | None, frequencies: Tensor, *,
           interleaved: bool = False, magnitude: float = 1.0) -> tuple[Tensor | None, Tensor | None]:
    """q [B, N, H, D] and k [B, N, Hk, D] (bf16 or fp32, strides as they come) turned to their positions.

    The first ``2 * len(frequencies)`` values of a head are taken as pairs (a, b): values i and i + len(frequencies), or
    2 i and 2 i + 1 (``interleaved``).  With t = position * frequency: a' = magnitude (a cos t - b sin t), b' =
    magnitude (a sin t + b cos t).  The rest of the head is left alone.
    positions: whole numbers that 32 bits hold [B, N] (None: 0, 1, ...); frequencies: 64 bits (``rotary_frequencies``).
    Either of q and k may be None, and is then None in the result.  D is a multiple of 8 up to 512.  Angles are computed
    in 64 bits: no position is too far.  Gradients: q and k."""
    like = k if q is None else q
    if like is None:
        raise ValueError("rotary: neither q nor k")
    _ops.require_gpu(like, "rotary")
    out = torch_op("rotary")(q, k, None if positions is None else _int32(positions, "rotary positions"), frequencies,
                             interleaved, magnitude, False)
    return (None if q is None else out[0]), (None if k is None else out[1])


class RotaryPosition(nn.Module):
    """``rotary`` with the frequencies of ``rotary_frequencies`` over the first ``dim`` values of a head; "parts" has the
    magnitude ``0.1 ln(factor) + 1`` unless another is given."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str | None = None,
                 factor: float = 1.0, length: int | None = None, turns: tuple[float, float] = (1.0, 32.0),
                 magnitude: float | None = None) -> None:
        super().__init__()
        self.dim, self.interleaved = dim, interleaved
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "parts" and factor > 1.0 else 1.0
        self.magnitude = magnitude
        # not a buffer: module.to(dtype) and half() would round it
        self._args = (dim, base, scaling, factor, length, turns)
        self.frequencies = self._make(None)

    def _make(self, device) -> Tensor:
        dim, base, scaling, factor, length, turns = self._args
        return rotary_frequencies(dim, base, scaling=scaling, factor=factor, length=length, turns=turns, device=device)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        device = fn(torch.empty(0, device=self.frequencies.device)).device
        # those of the meta device have no values to move (``to_empty``)
        self.frequencies = self._make(device) if self.frequencies.is_meta else self.frequencies.to(device)
        return self

    def forward(self, q: Tensor | None, k: Tensor | None = None,
                positions: Tensor | None = None) -> tuple[Tensor | None, Tensor | None]:
        return rotary(q, k, positions, self.frequencies, interleaved=self.interleaved, magnitude=self.magnitude)
