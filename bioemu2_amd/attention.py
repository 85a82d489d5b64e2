"""Attention over packed sequences and caches on MI355X, trainable.

``AttentionPairBias`` computes its bias from the pair representation, over one
padded batch, for inference.  ``attention`` takes q, k and v and serves what a
model over sequences needs beside it: many sequences packed into one row
(``segments``), causal and prefix masks, scores capped by a tanh, a learned bias
by buckets of distance, shared key/value heads, a cache with a length per
sequence (single tokens, or a few at a time), and the gradients of q, k, v and of
the bias table.  Keys that a query does not see have weight zero (not the large
negative score of ``AttentionPairBias``), and a query that sees none gives zeros.

Types as elsewhere: bf16, or fp32 under bf16 autocast, runs on bf16 operands with
fp32 accumulation; fp32 with autocast off in fp32.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from . import _ops
from ._lib import torch_op
from .paged_cache import PagedCache
from .relative_position import _int32, distance_buckets


def attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    scale: float | None = None,
    cap: float | None = None,
    bias_table: Tensor | None = None,
    bias_buckets: Tensor | None = None,
    segments: Tensor | None = None,
    key_segments: Tensor | None = None,
    causal: bool = False,
    prefix: Tensor | None = None,
    cache_lengths: Tensor | None = None,
) -> Tensor:
    """[B, Nq, H, D]: softmax over the keys that query i sees of ``cap tanh(scale q_i.k_j / cap) + bias``, times v.

    q: [B, Nq, H, D]; k, v: [B, Nk, Hk, D], H a multiple of Hk; D a multiple of 8 up to 128; bf16 or fp32, strides as
    they come.  The queries are the last Nq of ``cache_lengths[b]`` positions (default Nk): p_i = length - Nq + i.
    Keys at or past the length are not seen, whatever they hold.

    scale: D ** -0.5 by default.  cap: none by default; at most 1e5 (in bf16 scores are off by 2e-7 of it up to 4096,
    by fp32 rounding beyond).
    bias_table ([num_buckets, H], fp32 or bf16) and bias_buckets (``distance_buckets``, radius at most 512): the bias is
    ``bias_table[bias_buckets[clamp(j - p_i, -radius, radius) + radius], h]``.
    segments ([B, Nq] whole numbers of 32 bits): a query sees keys of its own segment only, and a negative one
    (padding) neither sees nor is seen, whatever it holds; key_segments ([B, Nk]) where the keys are others.  Values
    that a query does not see for another reason have to be finite; one that is not, where it is seen, reaches the result
    (in fp32 an infinity as NaN).
    causal: only keys j <= p_i, and those below ``prefix[b]`` ([B] whole numbers; nothing to say without causal)."""
    _ops.require_gpu(q, "attention")
    if q.ndim != 4:
        raise ValueError(f"attention: q must be [B, Nq, H, D], got {tuple(q.shape)}")
    if key_segments is None:
        key_segments = segments
    elif segments is None:
        raise ValueError("attention: segments of queries and of keys come together")
    if segments is not None:
        same = key_segments is segments
        segments = _int32(segments, "attention segments")
        key_segments = segments if same else _int32(key_segments, "attention key segments")
    if prefix is not None:
        prefix = _int32(prefix, "attention prefix")
    if cache_lengths is not None:
        cache_lengths = _int32(cache_lengths, "attention cache_lengths")
    if cap is not None and not cap > 0:
        raise ValueError(f"attention: cap must be positive, got {cap}")
    dtype = q.dtype
    if dtype == torch.float32 and not _ops.fp32_mode(q):
        q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    out = torch_op("attention")(
        q, k, v, bias_table, bias_buckets, segments, key_segments, prefix, cache_lengths,
        q.shape[-1] ** -0.5 if scale is None else scale, 0.0 if cap is None else cap, causal)
    return out if out.dtype == dtype else out.to(dtype)


class SequenceAttention(nn.Module):
    """``attention`` with a learned bias by buckets of distance (``distance_buckets(radius, num_buckets)``, one value
    per bucket and head) and fixed scale, cap and causality."""

    def __init__(self, num_heads: int, radius: int = 32, num_buckets: int | None = None, scale: float | None = None,
                 cap: float | None = None, causal: bool = False) -> None:
        super().__init__()
        buckets = distance_buckets(radius, num_buckets)
        self.num_heads, self.scale, self.cap, self.causal = num_heads, scale, cap, causal
        self.register_buffer("buckets", buckets, persistent=False)
        self.bias = nn.Parameter(torch.zeros(int(buckets.max()) + 1, num_heads))

    def forward(self, q: Tensor, k: Tensor, v: Tensor, segments: Tensor | None = None,
                key_segments: Tensor | None = None, prefix: Tensor | None = None,
                cache_lengths: Tensor | None = None) -> Tensor:
        return attention(q, k, v, scale=self.scale, cap=self.cap, bias_table=self.bias, bias_buckets=self.buckets,
                         segments=segments, key_segments=key_segments, causal=self.causal, prefix=prefix,
                         cache_lengths=cache_lengths)

    def paged(self, q: Tensor, cache: PagedCache, page_table: Tensor, lengths: Tensor,
              counts: Tensor | None = None) -> Tensor:
        """The same of new tokens over a cache in pages (``paged_attention``; no gradients)."""
        return cache.attend(q, page_table, lengths, counts=counts, scale=self.scale, cap=self.cap,
                            bias_table=self.bias.detach(), bias_buckets=self.buckets, causal=self.causal)
