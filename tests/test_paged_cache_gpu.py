"""Appending to a paged cache and attention over it against float64.

Tolerances, with u = 2^-24 and h = half a step of the type (2^-8 of a value in bf16, 2^-24 in fp32):
  e   a score's error in natural units: its D products are added in fp32, (D + 8) u scale sum|q||k|, 8 u of the score
      itself and of the bias, and 4e-7 cap for the tanh.  A weight is off by 2 e + 2 n u of itself (its own score and the
      row's sum, over n keys), and in bf16 by 2^-16 for its two parts.
  o   (w + 2 e + 4 n u) sum p|v| with w = 2^-16 (bf16) or u, and h of the result.  A weight below 2^-126 may be 0:
      2^-100 more.
Appended values are copied bit for bit; appended keys and the returned q are off as derived for rotary positions: 8 u +
2^-51 t of (|a| + |b|) and half a step of the result.
"""

from __future__ import annotations

import math
import threading

import pytest
import torch

from bioemu2_amd._lib import torch_op
from bioemu2_amd.attention import SequenceAttention, attention
from bioemu2_amd.paged_cache import PagedCache, paged_append, paged_attention
from bioemu2_amd.relative_position import distance_buckets
from bioemu2_amd.rotary import RotaryPosition, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    """Sequences of the given lengths in pages of any order; NaN wherever no sequence stands."""

    def __init__(self, lengths, dtype=BF16, Nq=1, H=4, Hk=2, D=32, page=16, counts=None, cap=None, radius=None,
                 num_buckets=None, tdtype=None, causal=True, scale=None, slots_first=False, width=None, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g) * spread).to(dtype).cuda()  # noqa: E731
        B = len(lengths)
        self.H, self.Hk, self.D, self.page = H, Hk, D, page
        self.q = rand(B, Nq, H, D)
        used = [-(-max(n, 0) // page) for n in lengths]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g).tolist()
        width = max([1, *used]) if width is None else width
        table = torch.full((B, width), -1, dtype=I32)
        shape = (pages, page, Hk, D) if slots_first else (pages, Hk, page, D)
        self.keys, self.values = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in "kv")
        if not slots_first:
            self.keys, self.values = self.keys.transpose(1, 2), self.values.transpose(1, 2)
        self.dense = []
        at = 0
        for b, n in enumerate(lengths):
            own = torch.tensor(order[at:at + used[b]], dtype=torch.long)
            at += used[b]
            table[b, :used[b]] = own[:width].to(I32)
            k, v = rand(n, Hk, D), rand(n, Hk, D)
            j = torch.arange(n)
            self.keys[own[j // page].cuda(), (j % page).cuda()] = k
            self.values[own[j // page].cuda(), (j % page).cuda()] = v
            self.dense.append((k, v))
        self.table = table.cuda()
        self.lengths = torch.tensor(lengths, dtype=I32).cuda()
        self.counts = None if counts is None else torch.tensor(counts, dtype=I32).cuda()
        self.cap, self.causal, self.scale = cap, causal, scale
        self.bias = self.buckets = None
        if radius is not None:
            self.buckets = distance_buckets(radius, num_buckets, device="cuda")
            self.bias = torch.randn(int(self.buckets.max()) + 1, H, generator=g).to(tdtype or dtype).cuda()

    def call(self, **over):
        kw = dict(counts=self.counts, scale=self.scale, cap=self.cap, bias_table=self.bias, bias_buckets=self.buckets,
                  causal=self.causal) | over
        return paged_attention(self.q, self.keys, self.values, self.table, self.lengths, **kw)

    def exact(self, hidden=None):
        """(value, bound); hidden[b]: truth values over the keys that are not to be seen."""
        B, Nq, H, D = self.q.shape
        G = H // self.Hk
        h = _half(self.q.dtype)
        w = 2.0 ** -16 if self.q.dtype == BF16 else U
        scale = D ** -0.5 if self.scale is None else self.scale
        value, bound = (torch.zeros(B, Nq, H, D, dtype=F64, device="cuda") for _ in "vb")
        for b, (k, v) in enumerate(self.dense):
            n = k.shape[0]
            count = Nq if self.counts is None else min(max(int(self.counts[b]), 0), Nq)
            if n == 0 or count == 0:
                continue
            k, v = (t.double().transpose(0, 1).repeat_interleave(G, 0) for t in (k, v))     # [H, n, D]
            q = self.q[b, :count].double().transpose(0, 1)                                   # [H, count, D]
            j, pos = torch.arange(n, device="cuda"), n - count + torch.arange(count, device="cuda")[:, None]
            ok = (j <= pos) if self.causal else torch.ones(count, n, dtype=torch.bool, device="cuda")
            if hidden is not None and hidden[b] is not None:
                ok = ok & ~hidden[b]
            k, v = (torch.where(ok.any(0)[:, None], t, 0.0) for t in (k, v))
            s = q @ k.transpose(1, 2) * scale
            e = (D + 8) * U * (q.abs() @ k.abs().transpose(1, 2)) * abs(scale)
            if self.cap:
                s = self.cap * torch.tanh(s / self.cap)
                e = e + 4e-7 * self.cap
            if self.bias is not None:
                r = self.buckets.numel() // 2
                bias = self.bias.double()[self.buckets.long()[(j - pos).clamp(-r, r) + r]].permute(2, 0, 1)
                s = s + bias
                e = e + 8 * U * bias.abs()
            e = 2 * torch.where(ok, e + 8 * U * s.abs(), 0.0).amax(-1, keepdim=True) + 4 * n * U + w
            p = torch.softmax(s.masked_fill(~ok, -math.inf), -1).nan_to_num(0.0)
            o = p @ v
            value[b, :count] = o.transpose(0, 1)
            bound[b, :count] = (e * (p @ v.abs()) + h * o.abs() + 2.0 ** -100).transpose(0, 1)
        return value, bound

    def check(self, got=None, **kw):
        got = self.call() if got is None else got
        value, bound = self.exact(**kw)
        off = (got.double() - value).abs()
        assert got.dtype == self.q.dtype and got.shape == value.shape and bool((off <= bound).all()), (
            float(off.max()), float((off / (bound + 1e-300)).max()))


WIDTHS = [(4, 2, 8), (3, 3, 24), (16, 16, 32), (8, 1, 40), (4, 4, 64), (6, 2, 80), (8, 2, 128), (17, 1, 128), (32, 1, 64), (40, 1, 24)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,Hk,D", WIDTHS)
def test_widths(gpu_device, dtype, H, Hk, D):
    Case([1, 2, 16, 33, 100, 0, 64], dtype, H=H, Hk=Hk, D=D).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 20, 32, 64, 100, 1000])
@pytest.mark.parametrize("slots_first", [False, True])
def test_pages(gpu_device, dtype, page, slots_first):
    Case([1, 31, 32, 33, 95, 200, 0], dtype, page=page, slots_first=slots_first, D=64).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kw", [dict(cap=5.0), dict(radius=8), dict(radius=40, num_buckets=32, cap=20.0), dict(scale=-0.3),
                                dict(radius=3, tdtype=F32), dict(cap=1e5), dict(causal=False, radius=8)], ids=str)
@pytest.mark.parametrize("Nq", [1, 5])
def test_scores(gpu_device, dtype, kw, Nq):
    Case([5, 40, 150, 77], dtype, Nq=Nq, H=8, Hk=2, D=64, **kw).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Nq,H,Hk", [(4, 4, 4), (4, 8, 2), (7, 9, 3), (16, 4, 2), (33, 2, 2), (40, 8, 2), (130, 3, 1)])
def test_few_queries_of_unequal_rows(gpu_device, dtype, causal, Nq, H, Hk):
    """Rows about one and two operands and several blocks; padding rows give zeros, whatever they hold."""
    c = Case([Nq, 150, 70, Nq + 1, 0, 1], dtype, Nq=Nq, H=H, Hk=Hk, D=32, counts=[Nq, max(1, Nq // 2), 0, Nq + 9, 0, 1],
             causal=causal)
    c.q[1, max(1, Nq // 2):] = math.nan
    c.check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths", [[1100], [5000], [1, 3000, 0, 40, 1025], [2000] * 9, [0, 0, 1500, 0], [0, 0]], ids=str)
@pytest.mark.parametrize("kw", [dict(), dict(Nq=3, cap=9.0, radius=100), dict(H=17, Hk=1, D=128), dict(Nq=12, H=8, Hk=2, page=20)], ids=str)
def test_keys_shared_out(gpu_device, dtype, lengths, kw):
    """Past 1024 keys of room the keys of all sequences are dealt to the workgroups and joined."""
    Case(lengths, dtype, width=None if max(lengths) > 1024 else 80, counts=None if kw.get("Nq", 1) == 1 else
         [min(n, kw["Nq"]) for n in lengths], **kw).check()


def test_many_sequences(gpu_device):
    """More sequences than a wave has lanes, some empty, in both plans."""
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 400, (150,), generator=g).tolist()
    lengths[:3], lengths[64], lengths[-1] = [0, 0, 0], 0, 0
    Case(lengths, H=4, Hk=2).check()
    Case(lengths, H=4, Hk=2, width=90).check()
    Case(lengths, H=8, Hk=8, width=90).check()          # more items than workgroups that share them
    Case(lengths * 4, H=8, Hk=8, D=16, width=90).check()   # so many that none is split


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,keys", [(43, 6, 20), (73, 7, 90), (37, 7, 9)])
def test_more_walks_than_units(gpu_device, dtype, B, H, keys):
    Case([1 + i * keys % 97 % keys for i in range(B)], dtype, H=H, Hk=H, D=64, radius=8).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("slots_first", [False, True])
def test_long_walks_of_narrow_heads(gpu_device, dtype, slots_first):
    Case([17011, 40], dtype, H=16, Hk=16, D=24, slots_first=slots_first).check()
    Case([17011, 0, 9000, 15], dtype, H=16, Hk=8, D=32, page=20, radius=100, slots_first=slots_first).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,Hk,Nq", [(1, 1, 1), (40, 1, 1), (12, 2, 3), (9, 3, 11)])
@pytest.mark.parametrize("radius,num_buckets", [(0, None), (127, None), (512, 256), (300, 8)])
def test_bias_tables(gpu_device, dtype, H, Hk, Nq, radius, num_buckets):
    Case([1100, 3, 300], dtype, H=H, Hk=Hk, Nq=Nq, radius=radius, num_buckets=num_buckets, tdtype=F32).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,D,most", [(24, 64, 3000), (48, 24, 2500), (64, 32, 1500), (65, 64, 1500), (33, 128, 1100)])
def test_parts_of_unequal_lengths(gpu_device, dtype, B, D, most):
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, most, (B,), generator=g).tolist()
    lengths[B // 2], lengths[1] = most, 0
    Case(lengths, dtype, H=8, Hk=8, D=D).check()


def test_one_long_sequence(gpu_device):
    for dtype in (BF16, F32):
        Case([70001], dtype, H=2, Hk=1, D=64, page=64).check()


def test_lengths_beyond_the_table_and_below_zero(gpu_device):
    c = Case([64, 64, 40], page=16)
    c.lengths.copy_(torch.tensor([10 ** 9, 64, -5]))
    # a length past the table is taken as the table's: position and distance with it
    c.dense[2] = (c.dense[2][0][:0], c.dense[2][1][:0])
    c.check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [None, 200])
def test_entries_that_name_no_page(gpu_device, dtype, width):
    c = Case([64, 100, 32, 5], dtype, page=16, width=width)
    pages = c.keys.shape[0]
    c.table[0, 1], c.table[1, 0], c.table[1, 5] = -1, pages, 2 ** 31 - 1
    c.table[2, :] = -2 ** 31
    hidden = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in (64, 100, 32, 5)]
    hidden[0][16:32] = True
    hidden[1][:16] = True
    hidden[1][80:96] = True
    hidden[2][:] = True
    c.check(hidden=hidden)


def test_empty_pool_or_table(gpu_device):
    q = torch.randn(2, 1, 4, 32, device="cuda", dtype=BF16)
    some = torch.zeros(3, 16, 2, 32, device="cuda", dtype=BF16)
    lengths = torch.tensor([5, 7], dtype=I32, device="cuda")
    for keys, table in ((some[:0], torch.zeros(2, 3, dtype=I32, device="cuda")),
                        (some, torch.zeros(2, 0, dtype=I32, device="cuda"))):
        out = paged_attention(q, keys, keys, table, lengths)
        assert out.shape == q.shape and out.abs().max() == 0
        k = torch.ones(2, 1, 2, 32, device="cuda", dtype=BF16)
        assert paged_append(keys, keys.clone(), k, k, table, lengths) is None
    assert some.abs().max() == 0
    assert paged_attention(q[:0], some, some, torch.zeros(0, 3, dtype=I32, device="cuda"), lengths[:0]).shape == (0, 1, 4, 32)
    assert paged_attention(q[:, :0], some, some, torch.zeros(2, 3, dtype=I32, device="cuda"), lengths).shape == (2, 0, 4, 32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width", [None, 90])
def test_what_is_not_finite_reaches_its_rows_only(gpu_device, dtype, width):
    c = Case([90, 90], dtype, Nq=2, H=4, Hk=2, width=width)
    want = c.call()
    for store in (c.keys, c.values):
        page, slot = int(c.table[0, 89 // 16]), 89 % 16     # the last key: seen by the last query alone
        old = store[page, slot, 1].clone()
        store[page, slot, 1, 5] = math.nan
        got = c.call()
        store[page, slot, 1] = old
        seen = torch.zeros_like(want, dtype=torch.bool)
        seen[0, 1, 2:] = True
        if store is c.values:
            only = torch.zeros_like(seen)
            only[..., 5] = True
            seen &= only
        assert torch.equal(got[~seen], want[~seen]) and bool(got[seen].isnan().all())


def test_scores_far_apart(gpu_device):
    """Maxima that move by more than a weight can hold, up and down the keys."""
    for dtype in (BF16, F32):
        c = Case([300, 1500], dtype, H=2, Hk=2, D=32, spread=8.0)
        c.check()
        k = c.dense[1][0]
        assert k.abs().max() > 20


@pytest.mark.parametrize("width", [None, 90])
def test_lowest_bias(gpu_device, width):
    """A row whose keys all have the type's lowest bias averages them; one of -infinity sees nothing."""
    c = Case([40, 40], F32, H=2, Hk=2, D=32, radius=0, width=width)
    c.bias[:, 0], c.bias[:, 1] = torch.finfo(F32).min, -math.inf
    out = c.call()
    for b in range(2):
        mean = c.dense[b][1][:, 0].double().mean(0)
        assert (out[b, 0, 0].double() - mean).abs().max() < 100 * U
        assert out[b, 0, 1].abs().max() == 0


@pytest.mark.parametrize("page,slots_outside", [(64, False), (64, True), (60, False)])
def test_offsets_past_32_bits(gpu_device, page, slots_outside):
    """Pages beyond 2^32 bytes (and beyond 2^31 values) of a pool, or its slots 2^26 bytes apart and more."""
    pages, hk, d = 70400, 4, 128          # 4.3 GB in bf16
    shape = (page, pages, hk, d) if slots_outside else (pages, hk, page, d)
    keys, values = (torch.empty(shape, dtype=BF16, device="cuda").transpose(*((0, 1) if slots_outside else (1, 2)))
                    for _ in "kv")
    lengths = torch.tensor([150], dtype=I32, device="cuda")
    table = torch.tensor([[pages - 1, 3, pages - 300]], dtype=I32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(1, 150, hk, d, generator=g, device="cuda").to(BF16) for _ in "kv")
    q = torch.randn(1, 1, hk, d, generator=g, device="cuda").to(BF16)
    paged_append(keys, values, k, v, table, lengths)
    assert torch.equal(keys[pages - 1], k[0, :page]) and torch.equal(values[pages - 300, :150 - 2 * page], v[0, 2 * page:])
    got = paged_attention(q, keys, values, table, lengths)
    want = attention(q.float(), k.float(), v.float())
    assert (got.float() - want).abs().max() < 2.0 ** -8 * want.abs().max() + 1e-4


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(gpu_device, dtype):
    """Heads of a wider cache, every other slot, a table cut from a wider one, q of a projection."""
    c = Case([70, 20], dtype, page=16, H=4, Hk=2, D=32)
    want = c.call()
    wide = torch.full((*c.keys.shape[:2], 5, 64), math.nan, dtype=dtype, device="cuda")
    wide[:, :, 1:3, 8:40], wide[:, :, 3:5, 16:48] = c.keys, c.values
    k, v = wide[:, :, 1:3, 8:40], wide[:, :, 3:5, 16:48]
    table = torch.full((2, 11), 7, dtype=I32, device="cuda")
    table[:, 4:4 + c.table.shape[1]] = c.table
    qkv = torch.zeros(2, 1, 3, 4, 32, dtype=dtype, device="cuda")
    qkv[:, :, 1] = c.q
    got = paged_attention(qkv[:, :, 1], k, v, table[:, 4:4 + c.table.shape[1]], c.lengths.long())
    assert torch.equal(got, want)
    odd = torch.empty(2, 1, 4, 36, dtype=dtype, device="cuda")
    odd[..., 1:33] = c.q
    assert torch.equal(paged_attention(odd[..., 1:33], k, v, c.table, c.lengths), want)


def test_slots_far_apart(gpu_device):
    """Slots more than 2^27 bytes apart (pages of 16, all first slots, then all second ones, ...)."""
    pages, page, hk, d = 131200, 16, 4, 128          # 2.1 GB
    keys, values = (torch.empty(page, pages, hk, d, dtype=BF16, device="cuda").transpose(0, 1) for _ in "kv")
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(1, 40, hk, d, generator=g, device="cuda").to(BF16) for _ in "kv")
    q = torch.randn(1, 1, hk, d, generator=g, device="cuda").to(BF16)
    lengths, table = torch.tensor([40], device="cuda"), torch.tensor([[131000, 7, 131199]], device="cuda")
    paged_append(keys, values, k, v, table, lengths)
    got, want = paged_attention(q, keys, values, table, lengths), attention(q.float(), k.float(), v.float())
    assert (got.float() - want).abs().max() < 2.0 ** -8 * want.abs().max() + 1e-4


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_queries_than_positions(gpu_device, dtype):
    """Queries before the first position see nothing."""
    c = Case([3, 1, 40], dtype, Nq=6, H=4, Hk=2, counts=[5, 6, 6])
    c.check()
    assert c.call()[0, :2].abs().max() == 0


def test_shared_pages(gpu_device):
    """Two sequences with the same beginning in the same pages."""
    c = Case([48, 64], page=16, H=4, Hk=2)
    c.table[0, :2] = c.table[1, :2]
    k, v = c.dense[1]
    c.dense[0] = (torch.cat((k[:32], c.dense[0][0][32:])), torch.cat((v[:32], c.dense[0][1][32:])))
    c.check()


# ----------------------------------------------------------------------------
# Appending
# ----------------------------------------------------------------------------
def _turned(x, pos, f, interleaved, magnitude):
    """(value, bound) of x [n, heads, D] at positions [n]."""
    n, h = f.numel(), _half(x.dtype)
    t = (pos.double()[:, None] * f)[:, None]
    c, s = magnitude * t.cos(), magnitude * t.sin()
    xd = x.double()
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = xd[..., ia], xd[..., ib]
    out, bound = xd.clone(), torch.zeros_like(xd)
    off = (8 * U + 2.0 ** -51 * t.abs()) * magnitude * (a.abs() + b.abs())
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    bound[..., ia], bound[..., ib] = off + h * out[..., ia].abs(), off + h * out[..., ib].abs()
    return out, bound


def _close(got, want):
    value, bound = want
    assert bool(((got.double() - value).abs() <= bound + 1e-38).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,H,Hk,D,rot,page,slots_first", [
    (1, 4, 2, 32, 32, 16, False), (1, 16, 16, 24, 24, 1, True), (5, 7, 7, 80, 40, 20, False), (70, 8, 2, 128, 128, 64, True),
    (3, 4, 1, 512, 512, 8, False), (300, 2, 2, 16, 6, 100, False), (2, 5, 5, 64, 0, 16, False)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(gpu_device, dtype, N, H, Hk, D, rot, page, slots_first, interleaved):
    counts = [N, N // 2, 0, N + 3, N]
    lengths = [N, N + 37, 40, N + 5, N + page]
    g = torch.Generator().manual_seed(N + D)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    B = 5
    q, k, v = rand(B, N, H, D), rand(B, N, Hk, D), rand(B, N, Hk, D)
    used = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(used) + 1, generator=g)
    table = torch.full((B, max(used)), -1, dtype=I32)
    for b in range(B):
        table[b, :used[b]] = order[sum(used[:b]):sum(used[:b + 1])].to(I32)
    keys, values = rand(sum(used) + 1, page, Hk, D), rand(sum(used) + 1, page, Hk, D)
    if not slots_first:
        keys, values = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (keys, values))
    k0, v0 = keys.clone(), values.clone()
    f = rotary_frequencies(rot, device="cuda") if rot else None
    kw = dict(interleaved=interleaved, magnitude=1.5)
    got = paged_append(keys, values, k, v, table.cuda(), torch.tensor(lengths, device="cuda"),
                       counts=torch.tensor(counts, device="cuda"), q=q if rot else None, frequencies=f, **kw)
    assert rot or got is None
    for b in range(B):
        n = min(counts[b], N)
        pos = torch.arange(lengths[b] - n, lengths[b])
        at = (table[b][pos // page].long().cuda(), (pos % page).cuda())
        if rot:
            _close(got[b, :n], _turned(q[b, :n], pos.cuda(), f, interleaved, 1.5))
            assert n == N or got[b, n:].abs().max() == 0
            _close(keys[at], _turned(k[b, :n], pos.cuda(), f, interleaved, 1.5))
        else:
            assert torch.equal(keys[at], k[b, :n])
        assert torch.equal(values[at], v[b, :n])
        keys[at], values[at] = k0[at], v0[at]
    assert torch.equal(keys, k0) and torch.equal(values, v0)     # nothing else was written


def test_append_positions_that_the_table_does_not_hold(gpu_device):
    keys, values = (torch.zeros(4, 8, 1, 16, dtype=F32, device="cuda") for _ in "kv")
    table = torch.tensor([[0, -1, 4], [2 ** 31 - 1, 1, 2], [3, 3, 3], [-2 ** 31, -1, 3]], dtype=I32, device="cuda")
    lengths = torch.tensor([24, 12, 3, 2 ** 31 - 1], dtype=I32, device="cuda")
    k = torch.ones(4, 24, 1, 16, dtype=F32, device="cuda")
    counts = torch.tensor([24, 12, 9, 24], dtype=I32, device="cuda")
    f = rotary_frequencies(16, device="cuda")
    q = paged_append(keys, values, k, 2 * k, table, lengths, counts=counts, q=k, frequencies=f,
                     positions=torch.zeros(4, 24, dtype=I32, device="cuda"))
    want = torch.zeros(4, 8)
    want[0] = 1            # sequence 0: its first page; pages -1 and 4 are none
    want[1, :4] = 1        # sequence 1: slots 8 .. 11
    want[3, :3] = 1        # sequence 2: positions -6 .. 2, of which 0 .. 2
    assert torch.equal(keys[:, :, 0, 0].cpu(), want) and torch.equal(values[:, :, 0, 3].cpu(), 2 * want)
    assert torch.equal(q[2, :9], k[2, :9]) and q[2, 9:].abs().max() == 0


def test_append_given_positions_and_negative_counts(gpu_device):
    keys, values = (torch.zeros(2, 8, 2, 32, dtype=F32, device="cuda") for _ in "kv")
    k, v = torch.randn(2, 3, 2, 32, device="cuda"), torch.randn(2, 3, 2, 32, device="cuda")
    pos = torch.tensor([[100, 7, 10 ** 6], [1, 2, 3]], dtype=I32, device="cuda")
    f = rotary_frequencies(32, device="cuda")
    paged_append(keys, values, k, v, torch.tensor([[1], [0]], device="cuda"), torch.tensor([5, 5], device="cuda"),
                 counts=torch.tensor([3, -4], device="cuda"), frequencies=f, positions=pos)
    _close(keys[1, 2:5], _turned(k[0], pos[0], f, False, 1.0))
    assert torch.equal(values[1, 2:5], v[0]) and keys[0].abs().max() == 0 and keys[1, :2].abs().max() == 0


def test_append_bumps_versions(gpu_device):
    cache = PagedCache(2, 8, 2, 32, device="cuda")
    cache.keys.zero_()
    k = torch.randn(1, 1, 2, 32, device="cuda", dtype=BF16)
    before = cache.keys._version, cache.values._version
    cache.append(k, k, torch.zeros(1, 1, dtype=I32, device="cuda"), torch.ones(1, dtype=I32, device="cuda"))
    assert cache.keys._version > before[0] and cache.values._version > before[1]
    before = cache.keys._version
    with torch.inference_mode():
        cache.append(k, k, torch.zeros(1, 1, dtype=I32, device="cuda"), torch.ones(1, dtype=I32, device="cuda"))
        own = PagedCache(2, 8, 2, 32, device="cuda")
        own.append(k, k, torch.zeros(1, 1, dtype=I32, device="cuda"), torch.ones(1, dtype=I32, device="cuda"))
    assert cache.keys._version > before


def test_append_of_the_cache_to_itself(gpu_device):
    """Slots moved by one within the cache: rows are read before they are written over."""
    cache = PagedCache(3, 16, 2, 32, dtype=F32, device="cuda")
    cache.keys.normal_()
    cache.values.normal_()
    k, v = cache.keys.clone(), cache.values.clone()
    table = torch.tensor([[0, 1]], dtype=I32, device="cuda")
    cache.append(cache.keys[:1, :15], cache.values[:1, :15], table, torch.tensor([16], device="cuda"))
    assert torch.equal(cache.keys[0, 1:], k[0, :15]) and torch.equal(cache.values[0, 1:], v[0, :15])
    assert torch.equal(cache.keys[0, 0], k[0, 0]) and torch.equal(cache.keys[1:], k[1:])


def test_append_past_the_caches(gpu_device):
    """More results than the caches near the CUs hold are written another way."""
    B, N, H, Hk, D, page = 2, 1500, 16, 16, 128, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(B, N, h, D, generator=g, device="cuda").to(BF16) for h in (H, Hk, Hk))
    cache = PagedCache(60, page, Hk, D, device="cuda")
    cache.keys.zero_()
    cache.values.zero_()
    table = torch.randperm(60, generator=torch.Generator().manual_seed(1))[:48].view(2, 24).to(I32)
    lengths, counts = [1533, 1400], [N, 1333]
    f = rotary_frequencies(D, device="cuda")
    got = cache.append(k, v, table.cuda(), torch.tensor(lengths, device="cuda"), counts=torch.tensor(counts, device="cuda"),
                       q=q, frequencies=f)
    for b in range(B):
        pos = torch.arange(lengths[b] - counts[b], lengths[b])
        at = (table[b][pos // page].long().cuda(), (pos % page).cuda())
        _close(got[b, :counts[b]], _turned(q[b, :counts[b]], pos.cuda(), f, False, 1.0))
        _close(cache.keys[at], _turned(k[b, :counts[b]], pos.cuda(), f, False, 1.0))
        assert torch.equal(cache.values[at], v[b, :counts[b]]) and bool((got[b, counts[b]:] == 0).all())
        cache.keys[at] = cache.values[at] = 0
    assert cache.keys.abs().max() == 0 and cache.values.abs().max() == 0


# ----------------------------------------------------------------------------
# Together
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_then_tokens_as_one_pass(gpu_device, dtype):
    """Two sequences, prompts of unequal length in one padded call, then tokens one by one and three at a time, against
    ``rotary`` and ``attention`` over each whole sequence."""
    torch.manual_seed(3)
    H, Hk, D, total, cap = 8, 2, 64, [90, 61], 30.0
    turn = RotaryPosition(D, interleaved=True).cuda()
    buckets = distance_buckets(20, 16, device="cuda")
    bias = torch.randn(int(buckets.max()) + 1, H, device="cuda").to(dtype)
    data = [[torch.randn(1, n, h, D, device="cuda").to(dtype) for h in (H, Hk, Hk)] for n in total]
    want = []
    for q, k, v in data:
        q, k = turn(q, k)
        want.append(attention(q, k, v, causal=True, cap=cap, bias_table=bias, bias_buckets=buckets))
    cache = PagedCache(20, 16, Hk, D, dtype=dtype, device="cuda")
    table = torch.tensor([[3, 9, 1, 12, 7, 15], [0, 19, 4, 8, 2, 6]], dtype=I32, device="cuda")
    done = [0, 0]

    def step(new):
        width = max(new)
        batch = [torch.full((2, width, h, D), math.nan, device="cuda").to(dtype) for h in (H, Hk, Hk)]
        for b, n in enumerate(new):
            for t, src in zip(batch, data[b]):
                t[b, :n] = src[0, done[b]:done[b] + n]
            done[b] += n
        lengths, counts = (torch.tensor(x, dtype=I32, device="cuda") for x in (done, new))
        q = cache.append(batch[1], batch[2], table, lengths, counts=counts, q=batch[0], frequencies=turn.frequencies,
                         interleaved=True)
        out = cache.attend(q, table, lengths, counts=counts, cap=cap, bias_table=bias, bias_buckets=buckets)
        for b, n in enumerate(new):
            a, w = out[b, :n].float(), want[b][0, done[b] - n:done[b]].float()
            # the same rounded q, k and v in both; sum p|v| <= max|v|.  bf16: one side's weights are off by h, both
            # results by h.  fp32: per side 2 e <= 2 ((D + 8) 5 + 16 + 7 cap) u <= 1200 u for scores of sum|q||k| / 8 <= 5,
            # 8 and a cap of 30, and 4 n u <= 360 u: 3200 u in both
            assert bool(((a - w).abs() <= (3 * _half(dtype) + 3200 * U) * data[b][2].float().abs().max()).all())
            assert bool((out[b, n:] == 0).all())

    step([40, 17])
    for _ in range(4):
        step([1, 1])
    step([3, 0])
    step([3, 3])
    while done[0] < 90:
        step([1, 1] if done[1] < 61 else [1, 0])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sequence_attention_over_pages(gpu_device, dtype):
    """A trained module over a cache: its bias wants gradients, the call has none; a query that does is refused."""
    c = Case([70, 5, 33], dtype, Nq=3, counts=[3, 1, 2], cap=20.0, radius=8, num_buckets=8, tdtype=F32, scale=0.2)
    att = SequenceAttention(4, radius=8, num_buckets=8, scale=0.2, cap=20.0, causal=True).cuda()
    with torch.no_grad():
        att.bias.copy_(c.bias)
    cache = PagedCache(1, c.page, c.Hk, c.D, dtype=dtype, device="cuda")
    cache.keys, cache.values = c.keys, c.values
    out = att.paged(c.q, cache, c.table, c.lengths, c.counts)
    assert not out.requires_grad
    c.check(out)
    with pytest.raises(NotImplementedError, match="no backward pass"):
        att.paged(c.q.clone().requires_grad_(), cache, c.table, c.lengths, c.counts)


@pytest.mark.parametrize("width", [8, 100])
def test_same_bits_other_stream_and_replays(gpu_device, width):
    """A captured step replayed with other lengths and tables, against the eager one."""
    c = Case([70, 100, 33], Nq=1, H=8, Hk=2, D=64, width=width)
    f = rotary_frequencies(64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(3, 1, 2, 64, generator=g, device="cuda").to(BF16) for _ in "kv")

    def step():
        q = paged_append(c.keys, c.values, k, v, c.table, c.lengths, q=c.q, frequencies=f)
        return paged_attention(q, c.keys, c.values, c.table, c.lengths)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    for lengths in ([70, 100, 33], [1, 1, 1], [64, 0, 40], [70, 99, 33]):
        c.lengths.copy_(torch.tensor(lengths))
        c.table.copy_(c.table.roll(1, 0) if lengths[0] == 64 else c.table)
        graph.replay()
        torch.cuda.synchronize()
        # as bits: a table that has moved on leads to slots that hold NaN
        assert torch.equal(out.view(torch.int16), step().view(torch.int16))


def test_two_graphs_do_not_share_space(gpu_device):
    cases = [Case([3000, 70, 2000], H=8, Hk=2, D=64, seed=s) for s in (1, 2)]
    want = [c.call() for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c, s in zip(cases, streams):
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(c.call())
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()
        torch.cuda.synchronize()


def test_two_threads_at_once(gpu_device):
    cases = [Case([2500, 60, 1300], dt, H=8, Hk=2, D=64, seed=i) for i, dt in enumerate((BF16, F32))]
    want = [c.call() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(c, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(c.call(), w):
                    bad.append(1)

    threads = [threading.Thread(target=work, args=x) for x in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_fp32_under_autocast(gpu_device):
    c = Case([40, 9], H=4, Hk=2)
    want = c.call()
    f = rotary_frequencies(32, device="cuda")
    k = torch.randn(2, 1, 2, 32, device="cuda")
    with torch.autocast("cuda", dtype=BF16):
        got = paged_attention(c.q.float(), c.keys, c.values, c.table, c.lengths)
        assert got.dtype == F32 and torch.equal(got, want.float())
        q = paged_append(c.keys, c.values, k, k, c.table, c.lengths, q=c.q.float(), frequencies=f)
    assert q.dtype == F32
    page, slot = int(c.table[0, 39 // 16]), 39 % 16
    assert torch.equal(c.values[page, slot], k[0, 0].to(BF16))
    with pytest.raises(ValueError, match="expected"):
        paged_attention(c.q.float(), c.keys, c.values, c.table, c.lengths)


@pytest.mark.parametrize("seed", range(40))
def test_arguments_in_any_combination(gpu_device, seed):
    import random

    r = random.Random(seed)
    Hk = r.choice([1, 1, 2, 3, 8])
    Nq = r.choice([1, 1, 2, 5, 20])
    lengths = [r.choice([0, 1, r.randint(1, 64), r.randint(1, 2500)]) for _ in range(r.randint(1, 7))]
    Case(lengths, r.choice([BF16, F32]), Nq=Nq, Hk=Hk, H=Hk * r.choice([1, 2, 5, 16]),
         D=r.choice([8, 16, 24, 32, 48, 64, 72, 96, 128]), page=r.choice([1, 2, 7, 16, 32, 48, 64, 128]),
         counts=[r.randint(0, min(Nq, n)) for n in lengths], cap=r.choice([None, 2.0, 50.0]),
         radius=r.choice([None, 5, 127]), causal=r.random() < 0.7, slots_first=r.random() < 0.5,
         width=r.choice([None, 2600]), seed=seed).check()


def test_fake_tensors(gpu_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, keys = (torch.empty(2, 1, 4, 32, dtype=BF16, device="cuda"), torch.empty(9, 16, 2, 32, dtype=BF16, device="cuda"))
        ints = torch.empty(2, 3, dtype=I32, device="cuda")
        out = torch_op("paged_attention")(q, keys, keys, ints, ints[:, 0], None, None, None, 1.0, 0.0, True)
        assert out.shape == q.shape and out.dtype == BF16
        out = torch_op("paged_append")(keys, keys, q[:, :, :2], q[:, :, :2], ints, ints[:, 0], None, q,
                                       torch.empty(16, dtype=F64, device="cuda"), None, False, 1.0)
        assert out.shape == q.shape


def test_refusals(gpu_device):
    c = Case([40, 9], H=4, Hk=2, D=32)
    good = dict(q=c.q, keys=c.keys, values=c.values, page_table=c.table, lengths=c.lengths)
    for over in [dict(q=c.q[0]), dict(q=c.q[..., :16]), dict(q=c.q[:, :, :3]), dict(q=c.q.float()), dict(q=c.q[:1]),
                 dict(keys=c.keys.float()), dict(keys=c.keys[:2]), dict(values=c.values[..., :16]), dict(keys=c.keys.cpu()),
                 dict(page_table=c.table.float()), dict(page_table=c.table[0]), dict(page_table=c.table.cpu()),
                 dict(lengths=c.lengths[:1]), dict(lengths=c.lengths.cpu()), dict(counts=c.lengths[:1]), dict(cap=0.0),
                 dict(cap=-1.0), dict(cap=2e5), dict(scale=math.nan), dict(bias_table=torch.zeros(3, 4, device="cuda")),
                 dict(bias_table=torch.zeros(3, 5, device="cuda"), bias_buckets=distance_buckets(1, device="cuda")),
                 dict(keys=c.keys.transpose(2, 3).contiguous().transpose(2, 3)),
                 dict(keys=c.keys[:, :0], values=c.values[:, :0]),
                 dict(page_table=torch.zeros(2, 1 << 24, dtype=I32, device="cuda"))]:
        with pytest.raises(ValueError):
            paged_attention(**(good | over))
    with pytest.raises(RuntimeError, match="no backward pass"):
        paged_attention(**(good | dict(q=c.q.clone().requires_grad_())))
    with torch.no_grad():
        paged_attention(**(good | dict(q=c.q.clone().requires_grad_())))
    f = rotary_frequencies(32, device="cuda")
    k = torch.zeros(2, 1, 2, 32, dtype=BF16, device="cuda")
    good = dict(keys=c.keys, values=c.values, k=k, v=k, page_table=c.table, lengths=c.lengths)
    before = c.keys.clone()
    for over in [dict(k=k[0]), dict(v=k[:, :, :1]), dict(k=k.float(), v=k.float()), dict(q=c.q), dict(positions=c.table[:, :1]),
                 dict(q=c.q.float(), frequencies=f), dict(q=c.q, frequencies=f.float()), dict(q=c.q, frequencies=f.repeat(2)),
                 dict(q=c.q[:1], frequencies=f), dict(frequencies=f, positions=c.table), dict(frequencies=f.cpu()),
                 dict(keys=c.keys[:1].expand(c.keys.shape)), dict(values=c.values[:, :1].expand(c.values.shape)),
                 dict(counts=c.lengths[:1]), dict(lengths=c.lengths.double())]:
        with pytest.raises(ValueError):
            paged_append(**(good | over))
    with pytest.raises(RuntimeError, match="no backward pass"):
        paged_append(**(good | dict(k=k.clone().requires_grad_())))
    assert torch.equal(c.keys.view(torch.int16), before.view(torch.int16))
