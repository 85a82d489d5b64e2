"""A cache of keys and values in pages on MI355X: appending to it and attending over it, for serving.

``attention`` reads one tensor of keys a sequence, which has to have room for the
longest.  Here sequences share a pool of pages of ``page_size`` slots, and a table
names each sequence's: ``keys`` and ``values`` are [pages, page_size, Hk, D],
position p of sequence b is slot ``p % page_size`` of page
``page_table[b, p // page_size]``.  A page may belong to several sequences (a shared
beginning), as long as nobody appends to it.  ``paged_append`` puts new keys and
values there, with rotary positions applied on the way; ``paged_attention`` is
``attention`` of the newest tokens over what is there.

Both take ``lengths`` (positions in use with the new ones) and, for batches of
unequal rows, ``counts`` (how many of them are new: row i of sequence b is position
``lengths[b] - counts[b] + i``, and rows from ``counts[b]`` on are padding).  Table,
lengths and counts are read on the GPU only, so a captured graph can be replayed
with other values in them.  They are of 32 bits; of 64 they are taken to the nearest
number of 32, two small kernels for each.  No gradients.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _ops
from ._lib import torch_op
from .relative_position import _int32


def _nearest_int32(t: Tensor, what: str) -> Tensor:
    """Whole numbers as the nearest of 32 bits: an entry of 2^32 is past any pool, not the first page."""
    if t.dtype == torch.int32:
        return t
    if t.dtype in (torch.uint32, torch.uint64):
        t = t.to(torch.int64)
    if t.dtype != torch.int64:
        return _int32(t, what)
    return t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _ints(what: str, page_table: Tensor, lengths: Tensor, counts: Tensor | None):
    return (_nearest_int32(page_table, f"{what} page_table"), _nearest_int32(lengths, f"{what} lengths"),
            None if counts is None else _nearest_int32(counts, f"{what} counts"))


def paged_append(keys: Tensor, values: Tensor, k: Tensor, v: Tensor, page_table: Tensor, lengths: Tensor, *,
                 counts: Tensor | None = None, q: Tensor | None = None, frequencies: Tensor | None = None,
                 positions: Tensor | None = None, interleaved: bool = False, magnitude: float = 1.0) -> Tensor | None:
    """Writes k and v ([B, N, Hk, D]) into the pages, in place, and returns q ([B, N, H, D]) turned like k (None without).

    keys, values: [pages, page_size, Hk, D] of k's type (bf16 or fp32; bf16 also for fp32 under bf16 autocast), values of
    a head adjacent, rows at 16-byte addresses, the other dimensions in any order in memory, no two slots in the same place
    (parts of one tensor may lie between each other if their strides are alike).  page_table: whole numbers of 32 bits
    [B, width]; lengths, counts: [B].  With ``frequencies`` k and q are turned as ``rotary`` does, to their
    positions in the sequence or to ``positions`` ([B, N], whole numbers that 32 bits hold).  Padding rows write nothing,
    and are zeros in the result; nor does a position whose table entry names no page (below 0, past the pool, or past the
    table).  A slot that a call names twice gets values of both, in any order.
    fp32 under bf16 autocast is rounded before it is turned, and again after: turn with ``rotary`` and append what it
    returns for one rounding."""
    _ops.require_gpu(k, "paged_append")
    page_table, lengths, counts = _ints("paged_append", page_table, lengths, counts)
    dtype = None if q is None else q.dtype
    if k.dtype == torch.float32 and keys.dtype == torch.bfloat16 and not _ops.fp32_mode(k):
        k, v, q = (None if t is None else t.to(torch.bfloat16) for t in (k, v, q))
    out = torch_op("paged_append")(
        keys, values, k, v, page_table, lengths, counts, q, frequencies,
        None if positions is None else _int32(positions, "paged_append positions"), interleaved, magnitude)
    return None if q is None else out.to(dtype)


def paged_attention(q: Tensor, keys: Tensor, values: Tensor, page_table: Tensor, lengths: Tensor, *,
                    counts: Tensor | None = None, scale: float | None = None, cap: float | None = None,
                    bias_table: Tensor | None = None, bias_buckets: Tensor | None = None, causal: bool = True) -> Tensor:
    """[B, Nq, H, D]: ``attention`` of q over the keys of each sequence's pages.

    q: [B, Nq, H, D] in the cache's type (or fp32 under bf16 autocast over a bf16 cache), H a multiple of the cache's Hk,
    D a multiple of 8 up to 128; row i of sequence b is at position ``lengths[b] - counts[b] + i`` (counts: Nq by
    default) and sees the keys up to its own (all of the sequence's, not causal); padding rows and rows that see nothing
    give zeros.  Made for a few rows a sequence: keys are read once for every 32 rows of queries times H / Hk (past some 256
    rows ``attention`` over keys laid side by side is faster, the copy included).
    Keys whose table entry names no page, or that the table does not reach, are not seen (positions count on past its
    end); what unused slots hold does not matter.
    Values that are not finite reach the rows that see them, and no others.
    scale, cap, bias_table, bias_buckets: as in ``attention``.  The table's width times the page size is at most 2^27, and
    times B Hk (and, past 32 rows, their blocks) below 2^35."""
    _ops.require_gpu(q, "paged_attention")
    if q.ndim != 4:
        raise ValueError(f"paged_attention: q must be [B, Nq, H, D], got {tuple(q.shape)}")
    if cap is not None and not cap > 0:
        raise ValueError(f"paged_attention: cap must be positive, got {cap}")
    page_table, lengths, counts = _ints("paged_attention", page_table, lengths, counts)
    dtype = q.dtype
    if dtype == torch.float32 and keys.dtype == torch.bfloat16 and not _ops.fp32_mode(q):
        q = q.to(torch.bfloat16)
    out = torch_op("paged_attention")(
        q, keys, values, page_table, lengths, counts, bias_table, bias_buckets,
        q.shape[-1] ** -0.5 if scale is None else scale, 0.0 if cap is None else cap, causal)
    return out if out.dtype == dtype else out.to(dtype)


class PagedCache:
    """One layer's pages, with the slots of a head side by side in memory (what ``paged_attention`` reads fastest)."""

    def __init__(self, pages: int, page_size: int, num_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device=None) -> None:
        shape = (pages, num_heads, page_size, head_dim)
        self.page_size = page_size
        self.keys = torch.empty(shape, dtype=dtype, device=device).transpose(1, 2)
        self.values = torch.empty(shape, dtype=dtype, device=device).transpose(1, 2)

    def append(self, k: Tensor, v: Tensor, page_table: Tensor, lengths: Tensor, **kw) -> Tensor | None:
        """``paged_append`` to this cache."""
        return paged_append(self.keys, self.values, k, v, page_table, lengths, **kw)

    def attend(self, q: Tensor, page_table: Tensor, lengths: Tensor, **kw) -> Tensor:
        """``paged_attention`` over this cache."""
        return paged_attention(q, self.keys, self.values, page_table, lengths, **kw)
