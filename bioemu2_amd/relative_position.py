"""Learned relative positions on MI355X.

``relative_position`` makes (or adds to) the pair representation an embedding of
each pair's residue offset, by buckets, with one more bucket for pairs of
different chains: what ``PairwiseConditioning`` takes as its relative-position
features and the trunk adds to its initial pair representation (the reference
computes them in ``biomoa/modules/relative_position_encoder.py``).  The table
has a gradient.  ``distance_buckets`` lays out the map from offsets to buckets,
which ``attention`` takes too.
"""

from __future__ import annotations

import bisect
import math
from fractions import Fraction

import torch
import torch.nn as nn
from torch import Tensor

from . import _ops
from ._lib import torch_op


def distance_buckets(radius: int, num_buckets: int | None = None, device=None) -> Tensor:
    """Buckets (uint8 [2 * radius + 1]) of the offsets -radius .. radius; offsets beyond count as the ends.

    Without ``num_buckets`` every offset has its own (2 * radius + 1 of them, at most 256).  With it (even), half of
    the buckets are for each direction (offset 0 among the positive ones): one per distance up to a quarter of them,
    the rest spaced logarithmically up to ``radius``.  The borders are found in whole numbers."""
    if radius < 0:
        raise ValueError(f"distance_buckets: radius {radius}")
    if num_buckets is None:
        if 2 * radius + 1 > 256:
            raise ValueError(f"distance_buckets: {2 * radius + 1} buckets, at most 256: give num_buckets")
        return torch.arange(2 * radius + 1, dtype=torch.uint8, device=device)
    if num_buckets % 4 or not 4 <= num_buckets <= 256:
        raise ValueError(f"distance_buckets: num_buckets must be a multiple of 4 up to 256, got {num_buckets}")
    half, exact = num_buckets // 2, num_buckets // 4
    if radius < exact:
        raise ValueError(f"distance_buckets: radius {radius} is below the {exact} exact distances")

    def first(k: int) -> int:
        """The least distance d of log bucket k: (d / exact) ** (half - exact) >= (radius / exact) ** k."""
        steps = half - exact
        d = max(exact, math.floor(exact * (radius / exact) ** (k / steps)) - 1)
        while Fraction(d, exact) ** steps < Fraction(radius, exact) ** k:
            d += 1
        return d

    borders = [first(k) for k in range(half - exact)]
    side = [d if d < exact else exact + bisect.bisect_right(borders, d) - 1 for d in range(radius + 1)]
    side = [min(b, half - 1) for b in side]
    return torch.tensor([half + b for b in side[:0:-1]] + side, dtype=torch.uint8, device=device)


def _int32(t: Tensor, what: str) -> Tensor:
    if t.dtype == torch.int32:
        return t
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise ValueError(f"{what}: expected whole numbers, got {t.dtype}")
    return t.to(torch.int32)


def relative_position(table: Tensor, buckets: Tensor, positions: Tensor, chains: Tensor | None = None,
                      z: Tensor | None = None, dtype: torch.dtype | None = None) -> Tensor:
    """[B, N, N, C]: ``table[bucket(positions[b, j] - positions[b, i])]``, the table's last row where ``chains``
    differ, added to ``z`` if given.

    table: [num_buckets, C] fp32 or bf16, at most 256 rows, C at most 4096 (256 where rows of the result are not whole
    16-byte pieces); buckets: uint8 [2 * radius + 1] (``distance_buckets``);
    positions, chains: whole numbers of 32 bits [B, N]; the result has z's type, or ``dtype`` (the table's by default), bf16 or
    fp32.  Gradients: ``table`` and ``z``."""
    _ops.require_gpu(table, "relative_position")
    if z is not None:
        if dtype is not None and dtype != z.dtype:
            raise ValueError(f"relative_position: dtype {dtype}, z is {z.dtype}")
        dtype = z.dtype
    return torch_op("relative_position")(
        table, z, buckets, _int32(positions, "relative_position positions"),
        None if chains is None else _int32(chains, "relative_position chains"), table.dtype if dtype is None else dtype)


class RelativePosition(nn.Module):
    """A learned embedding of residue offsets: ``dim`` channels for each bucket of ``distance_buckets(radius,
    num_buckets)`` and one bucket for pairs of different chains."""

    def __init__(self, dim: int, radius: int = 32, num_buckets: int | None = None) -> None:
        super().__init__()
        buckets = distance_buckets(radius, num_buckets)
        self.dim, self.radius = dim, radius
        self.num_buckets = int(buckets.max()) + 2   # the last one: different chains
        if self.num_buckets > 256:
            raise ValueError(f"RelativePosition: {self.num_buckets} buckets, at most 256")
        self.register_buffer("buckets", buckets, persistent=False)
        self.weight = nn.Parameter(torch.empty(self.num_buckets, dim))
        nn.init.normal_(self.weight, std=dim ** -0.5)

    def forward(self, positions: Tensor, chains: Tensor | None = None, z: Tensor | None = None,
                dtype: torch.dtype | None = None) -> Tensor:
        return relative_position(self.weight, self.buckets, positions, chains, z, dtype)
