"""Trainable LayerNorm on MI355X.

The inference modules of this package fold their LayerNorms into the products
that follow; a training step needs the normalised rows and their gradients.
``LayerNorm`` has ``torch.nn.LayerNorm``'s parameters and ``state_dict`` keys for
one normalised dimension; ``layer_norm`` is the function.  bf16 and fp32
activations, parameters in either; statistics and sums are fp32 and the weight
gradients deterministic.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from . import _ops
from ._lib import torch_op


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's type (bf16 or fp32).

    ``weight`` and ``bias`` ([c], fp32 or bf16, one type) may be absent.  Rows may have any stride; c is at most 16384
    where rows are whole 16-byte vectors and 4096 else."""
    _ops.require_gpu(x, "layer_norm")
    return torch_op("layer_norm")(x, weight, bias, eps)


class LayerNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True) -> None:
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if elementwise_affine and bias else None

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1] != self.dim:
            raise ValueError(f"LayerNorm: expected last dimension {self.dim}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
