"""Attention and its gradients against float64.

Tolerances, with u = 2^-24 and h = half a step of the operands' type (2^-8 of a value in bf16, 2^-24 in fp32):
  e   a score's error in natural units: its D products are added one after the other in fp32, (D + 8) u scale sum|q||k|,
      8 u of the score itself and of the bias, and 4e-7 cap for the tanh.  A weight is then off by 2 e + n u of itself
      (its own score and the row's sum), n the row's keys.
  do  (h + 2 e + 2 n u) sum p|v|, and half a step of the result.
  The row sum delta = do . o is off by w = sum_d |do| (off(o) + half a step of o) + D u sum|do||o|; dp by D u sum|do||v|:
  ds  p ((2 e + 2 n u) |dp - delta| + w + D u sum|do||v|) = E
  dq  scale sum_j (E + (h + 2e-6) |ds|) |k| + n u scale sum|ds||k|, and half a step;  dk the same over queries with |q|
  dv  sum_i (h + 2 e + 2 n u) p |do|, and half a step
  dtable  sum E + m u sum|ds| over the bucket's m pairs, and half a step
n counts the longest chain of fp32 adds, the keys (or queries) themselves.  A weight below 2^-126, fp32's least normal
number, may come out as 0: with n < 2^16 of them, each times values below 2^10 here, 2^-100 more of every result.
"""

from __future__ import annotations

import math

import pytest
import torch

from bioemu2_amd._lib import torch_op
from bioemu2_amd.attention import SequenceAttention, attention
from bioemu2_amd.layer_norm import LayerNorm
from bioemu2_amd.relative_position import RelativePosition, distance_buckets

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    def __init__(self, device, dtype=BF16, B=2, Nq=70, Nk=None, H=4, Hk=None, D=32, segments=None, causal=False,
                 prefix=None, lengths=None, cap=None, radius=None, num_buckets=None, tdtype=None, scale=None, seed=0,
                 spread=1.0):
        Nk = Nq if Nk is None else Nk
        Hk = H if Hk is None else Hk
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=g) * spread).to(dtype).to(device)  # noqa: E731
        self.q, self.k, self.v = rand(B, Nq, H, D), rand(B, Nk, Hk, D), rand(B, Nk, Hk, D)
        self.do = torch.randn(B, Nq, H, D, generator=g).to(dtype).to(device)
        self.causal, self.cap, self.scale = causal, cap, scale
        as_int = lambda t: None if t is None else torch.as_tensor(t, dtype=torch.int32).to(device)  # noqa: E731
        self.prefix, self.lengths = as_int(prefix), as_int(lengths)
        self.segments = self.key_segments = None
        if segments is not None:
            q_seg, k_seg = segments if isinstance(segments, tuple) else (segments, segments)
            self.segments, self.key_segments = as_int(q_seg), as_int(k_seg)
        self.table = self.buckets = None
        if radius is not None:
            self.buckets = distance_buckets(radius, num_buckets, device=device)
            self.table = torch.randn(int(self.buckets.max()) + 1, H, generator=g).to(tdtype or dtype).to(device)

    def call(self, **over):
        kw = dict(scale=self.scale, cap=self.cap, bias_table=self.table, bias_buckets=self.buckets,
                  segments=self.segments, key_segments=self.key_segments, causal=self.causal, prefix=self.prefix,
                  cache_lengths=self.lengths) | over
        return attention(self.q, self.k, self.v, **kw)

    def step(self):
        leaves = [t for t in (self.q, self.k, self.v, self.table) if t is not None]
        for t in leaves:
            t.requires_grad_(True)
        o = self.call()
        return [o.detach(), *torch.autograd.grad(o, leaves, self.do)]

    def allowed(self):
        B, Nq, _, _ = self.q.shape
        Nk, dev = self.k.shape[1], self.q.device
        j = torch.arange(Nk, device=dev)
        length = torch.full((B,), Nk, device=dev) if self.lengths is None else self.lengths.long().clamp(0, Nk)
        pos = (length - Nq)[:, None] + torch.arange(Nq, device=dev)
        ok = (j < length[:, None, None]).expand(B, Nq, Nk)
        if self.causal:
            seen = j <= pos[:, :, None]
            if self.prefix is not None:
                seen = seen | (j < self.prefix[:, None, None])
            ok = ok & seen
        if self.segments is not None:
            ok = ok & (self.segments[:, :, None] == self.key_segments[:, None, :]) & (self.segments[:, :, None] >= 0)
        return ok, pos, j

    def exact(self, train=True):
        """[(value, bound)] of o, dq, dk, dv and the table's gradient."""
        B, Nq, H, D = self.q.shape
        Nk, Hk = self.k.shape[1], self.k.shape[2]
        G, dtype = H // Hk, self.q.dtype
        ok, pos, j = self.allowed()
        ok = ok[:, None]
        clean = lambda t, seen: torch.where(seen[:, :, None, None], t.detach(), torch.zeros_like(t)).double()  # noqa: E731
        # what is not in play does not count, whatever it holds
        q, do = (clean(t, ok[:, 0].any(2)).transpose(1, 2).contiguous() for t in (self.q, self.do))
        k, v = (clean(t, ok[:, 0].any(1)).transpose(1, 2).repeat_interleave(G, 1).contiguous() for t in (self.k, self.v))
        kt, vt = k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous()
        scale = D ** -0.5 if self.scale is None else self.scale
        x = torch.matmul(q, kt) * scale
        size = torch.matmul(q.abs(), kt.abs()) * abs(scale)
        slope = torch.ones_like(x)
        s = x
        e = (D + 8) * U * size
        if self.cap:
            t = torch.tanh(x / self.cap)
            s, slope = self.cap * t, 1 - t * t
            e = e + 4e-7 * self.cap
        which = None
        if self.table is not None:
            R = self.buckets.numel() // 2
            which = self.buckets.long()[(j - pos[:, :, None]).clamp(-R, R) + R].clamp(max=self.table.shape[0] - 1)
            bias = self.table.detach().double()[which].permute(0, 3, 1, 2)
            s = s + bias
            # next to the type's lowest value nothing of a score is left: such keys are equal, or weigh nothing beside others
            low = bias < -1e30
            other = (ok & ~low).any(-1, keepdim=True)
            s = torch.where(low, torch.where(other, -math.inf, 0.0), s)
            e = torch.where(low, 0.0, e + 8 * U * bias.abs())
        e = e + 8 * U * torch.where(s == -math.inf, 0.0, s.abs())
        s = s.masked_fill(~ok, -math.inf)
        p = torch.where(ok.any(-1, keepdim=True), torch.softmax(s, -1), 0.0).nan_to_num(0.0)
        e = 2 * torch.where(ok, e, 0.0).amax(-1, keepdim=True) + 2 * Nk * U
        h = _half(dtype) if dtype == BF16 else U
        o = torch.matmul(p, v)
        off_o = (h + e) * torch.matmul(p, v.abs())
        back = lambda t: t.transpose(1, 2)  # noqa: E731
        res = [(back(o), back(off_o + h * o.abs()))]
        if not train:
            return res
        pT = p.transpose(2, 3).contiguous()
        fold = lambda t: t.view(B, Hk, G, Nk, D).sum(2)  # noqa: E731
        dv = fold(torch.matmul(pT, do))
        e_rows = (h + e) * p + 2 * Nq * U * p
        dv_off = fold(torch.matmul(e_rows.transpose(2, 3).contiguous(), do.abs())) + h * dv.abs()
        dp = torch.matmul(do, vt)
        w = (do.abs() * (off_o + h * o.abs())).sum(-1, keepdim=True) + D * U * (do.abs() * o.abs()).sum(-1, keepdim=True)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        E = p * (e * (dp - delta).abs() + w + D * U * torch.matmul(do.abs(), vt.abs()))
        table = None
        if which is not None:
            nb = self.table.shape[0]
            idx = which[:, None].expand(B, H, Nq, Nk) + nb * torch.arange(H, device=q.device)[:, None, None]
            fold_t = lambda t: torch.zeros(H * nb, dtype=F64, device=q.device).index_add_(  # noqa: E731
                0, idx.reshape(-1), t.reshape(-1)).view(H, nb).t()
            table = fold_t(ds)
            count = fold_t(ok.expand(B, H, Nq, Nk).double())
            table = (table, fold_t(E) + count * U * fold_t(ds.abs()) + _half(self.table.dtype) * table.abs())
        ds, E = ds * slope, E * slope + (h + 2e-6) * (ds * slope).abs() + (4e-6 * ds.abs() if self.cap else 0.0)
        dq = torch.matmul(ds, k) * scale
        dq_off = torch.matmul(E + Nk * U * ds.abs(), k.abs()) * abs(scale) + h * dq.abs()
        dsT, ET = ds.transpose(2, 3).contiguous(), (E + Nq * G * U * ds.abs()).transpose(2, 3).contiguous()
        dk = fold(torch.matmul(dsT, q)) * scale
        dk_off = fold(torch.matmul(ET, q.abs())) * abs(scale) + h * dk.abs()
        res += [(back(dq), back(dq_off)), (back(dk), back(dk_off)), (back(dv), back(dv_off))]
        return res + ([table] if table is not None else [])


def check(got, want, names=("o", "dq", "dk", "dv", "dtable")):
    assert len(got) == len(want)
    for g, (value, bound), name in zip(got, want, names):
        assert g.shape == value.shape and bool(g.isfinite().all()), name
        err = (g.double() - value).abs()
        bound = bound + 2.0 ** -100
        worst = (err - bound).max().item()
        print(f"{name}: off {err.max().item():.3e}, allowed {bound.max().item():.3e}, "
              f"share {(err / bound.clamp(min=1e-300)).max().item():.3f}", flush=True)
        assert worst <= 0, (name, worst)


def packed(B, N, lengths, hole=0):
    """Segment ids of `lengths` rows one after the other, `hole` rows of padding between them, padding behind."""
    row = []
    for s, n in enumerate(lengths):
        row += [s] * n + [-1] * hole
    row = (row + [-1] * N)[:N]
    return torch.tensor([row] * B)


SHAPES = [dict(B=1, Nq=1, H=1, D=8), dict(B=1, Nq=33, H=2, D=24), dict(B=2, Nq=70, H=4, D=32),
          dict(B=1, Nq=129, H=2, D=40), dict(B=2, Nq=200, H=4, D=64), dict(B=1, Nq=257, H=2, D=128),
          dict(B=1, Nq=65, H=3, D=96)]
MASKS = {
    "plain": dict(), "causal": dict(causal=True), "capped": dict(cap=2.0), "bias": dict(radius=8),
    "causal_bias_capped": dict(causal=True, radius=20, cap=5.0),
}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"n{s['Nq']}d{s['D']}")
def test_step(gpu_device, dtype, mask, shape):
    c = Case(gpu_device, dtype, **shape, **MASKS[mask])
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 64), (6, 1, 32), (4, 2, 128)])
@pytest.mark.parametrize("kw", [dict(), dict(causal=True, radius=16), dict(cap=3.0, causal=True, prefix=[40, 0])],
                         ids=["plain", "causal_bias", "prefix_capped"])
def test_shared_heads(gpu_device, dtype, H, Hk, D, kw):
    c = Case(gpu_device, dtype, B=2, Nq=150, H=H, Hk=Hk, D=D, **kw)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths,hole", [([1], 0), ([64, 64, 64], 0), ([5, 1, 90, 31, 2, 150], 0), ([30, 70, 40], 3),
                                          ([300], 0), ([], 0), ([1] * 40, 1)])
@pytest.mark.parametrize("kw", [dict(), dict(causal=True, radius=12, num_buckets=None), dict(causal=True, prefix=[9, 100])],
                         ids=["plain", "causal_bias", "prefix"])
def test_packed_sequences(gpu_device, dtype, lengths, hole, kw):
    c = Case(gpu_device, dtype, B=2, Nq=300, H=2, D=32, segments=packed(2, 300, lengths, hole), **kw)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_segments_in_any_order(gpu_device, dtype):
    g = torch.Generator().manual_seed(3)
    seg = torch.randint(-1, 4, (2, 190), generator=g)
    seg[1] = seg[1] * 1000000 + 7
    check(*(lambda c: (c.step(), c.exact()))(Case(gpu_device, dtype, B=2, Nq=190, H=2, D=64, segments=seg, radius=30)))
    k_seg = torch.randint(-1, 4, (2, 91), generator=g)
    check(*(lambda c: (c.step(), c.exact()))(
        Case(gpu_device, dtype, B=2, Nq=190, Nk=91, H=4, Hk=2, D=32, segments=(torch.randint(0, 4, (2, 190), generator=g), k_seg))))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 2), (1, 300), (1, 2000), (4, 777), (8, 31), (40, 333), (200, 900), (130, 60)])
@pytest.mark.parametrize("kw", [dict(causal=True), dict(), dict(causal=True, radius=33, cap=4.0)],
                         ids=["causal", "plain", "bias_capped"])
def test_cache(gpu_device, dtype, Nq, Nk, kw):
    """Lengths from nothing to the whole cache; queries before position 0 see nothing."""
    c = Case(gpu_device, dtype, B=4, Nq=Nq, Nk=Nk, H=8, Hk=2, D=64, lengths=[Nk, Nk // 2, min(1, Nk), 0], **kw)
    check([c.call().detach()], c.exact(train=False))
    check(c.step(), c.exact())


@pytest.mark.parametrize("D", [24, 32, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_single_tokens_of_other_widths(gpu_device, dtype, D):
    c = Case(gpu_device, dtype, B=3, Nq=1, Nk=1500, H=8, Hk=8, D=D, lengths=[1500, 700, 33], causal=True, radius=64, num_buckets=32)
    check([c.call().detach()], c.exact(train=False))
    c = Case(gpu_device, dtype, B=1, Nq=2, Nk=999, H=16, Hk=1, D=D, causal=True,
             segments=(torch.full((1, 2), 1), torch.arange(999)[None] // 500))
    check([c.call().detach()], c.exact(train=False))


def test_long_keys_split_and_joined(gpu_device):
    c = Case(gpu_device, BF16, B=1, Nq=50, Nk=6000, H=1, D=64, causal=True)
    check([c.call().detach()], c.exact(train=False))
    c = Case(gpu_device, BF16, B=1, Nq=50, Nk=6000, H=1, D=32, segments=(packed(1, 50, [20, 29]), packed(1, 6000, [2500, 2000])))
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kw", [dict(causal=True), dict(causal=True, cap=4.0, radius=30), dict()], ids=["causal", "bias_capped", "plain"])
def test_long_walks_in_parts(gpu_device, dtype, kw):
    """Walks long enough to be dealt to several workgroups beside those that fill the card."""
    c = Case(gpu_device, dtype, B=1, Nq=4133, H=2, Hk=1, D=24, **kw)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_longest_walks_of_wide_heads(gpu_device, dtype):
    """A few rows at the end of 8200 keys (the gradients of all of them), heads of 128."""
    c = Case(gpu_device, dtype, B=1, Nq=300, Nk=8200, H=2, Hk=2, D=128, causal=True)
    check(c.step(), c.exact())


def test_more_blocks_than_one_list(gpu_device):
    """More than 1024 blocks of 32 keys in fp32: the list of active blocks is made in two parts."""
    seg = packed(1, 34000, [200, 33000, 500])
    c = Case(gpu_device, F32, B=1, Nq=130, Nk=34000, H=1, D=8, segments=(torch.tensor([[0] * 40 + [1] * 40 + [2] * 45 + [-1] * 5]), seg))
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_padding_holds_does_not_count(gpu_device, dtype):
    """NaN and infinities in padded positions and past the length reach nothing, forward and backward."""
    seg = packed(2, 150, [40, 60], hole=5)
    c = Case(gpu_device, dtype, B=2, Nq=150, H=2, D=64, segments=seg, radius=16)
    pad = (seg < 0).to(gpu_device)
    want = c.step()
    for t, x in ((c.q, math.nan), (c.k, math.inf), (c.v, math.nan), (c.do, -math.inf)):
        t.data[pad] = x
    got = c.step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(bool((t[pad] == 0).all()) for t in got[:4])
    for Nq in (1, 60):
        c = Case(gpu_device, dtype, B=2, Nq=Nq, Nk=200, H=4, Hk=2, D=32, lengths=[90, 0], causal=True)
        c.k[0, 90:], c.v[0, 90:], c.k[1], c.v[1] = math.nan, math.inf, math.nan, math.nan
        check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lowest_values_and_infinities_as_bias(gpu_device, dtype):
    """A bias of -infinity hides its keys; the type's lowest value leaves a finite score (a row of such scores is an
    average)."""
    for value in (-math.inf, torch.finfo(dtype).min):
        c = Case(gpu_device, dtype, B=1, Nq=100, H=2, D=32, radius=3)
        c.table[:3] = value          # keys before the query
        o = c.call()
        ref = Case(gpu_device, dtype, B=1, Nq=100, H=2, D=32, radius=3)
        ref.table[:3] = -1e4
        want = ref.exact(train=False)
        check([o], want)
        c.table[:] = value
        o = c.call()
        if value == -math.inf:
            assert bool((o == 0).all())
        else:
            mean = c.v.double().mean(1, keepdim=True).expand(1, 100, 2, 32)
            assert bool(((o.double() - mean).abs() <= 2 * _half(dtype) * c.v.double().abs().mean(1, keepdim=True) + 200 * U * 5).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kw", [dict(), dict(causal=True), dict(causal=True, cap=3.0),
                                dict(causal=True, segments=packed(1, 200, [70, 100]))],
                         ids=["plain", "causal", "capped", "packed"])
def test_gradients_of_rows_at_the_lowest_bias(gpu_device, dtype, kw):
    """Keys within reach at the type's lowest value, those beyond ordinary: the first rows of a causal sequence see only
    the former and average them, with the gradients of an average; and one head at the lowest value throughout."""
    c = Case(gpu_device, dtype, B=1, Nq=200, H=4, Hk=2, D=32, radius=40, **kw)
    low = torch.finfo(dtype).min
    c.table[1:-1] = low
    c.table[:, 3] = low
    check(c.step(), c.exact())


def test_large_bias_and_lengths_off_a_tile(gpu_device):
    """Bias values whose exponential overflows: what stands behind the last query of a tile stays without weight."""
    for Nq in (33, 70, 130):
        c = Case(gpu_device, F32, B=1, Nq=Nq, H=2, D=32, radius=4)
        c.table += 150.0
        check(c.step(), c.exact())
        c.table.requires_grad_(False).mul_(40.0)
        check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_widest_bias_and_all_buckets(gpu_device, dtype):
    c = Case(gpu_device, dtype, B=1, Nq=1100, Nk=1150, H=2, Hk=1, D=128, radius=512, num_buckets=256, causal=True)
    assert c.table.shape[0] == 256
    check(c.step(), c.exact())


def test_more_query_blocks_than_one_list(gpu_device):
    """More than 1024 blocks of 32 queries in fp32: the keys' walk over the queries is listed in two parts."""
    seg = packed(1, 34000, [200, 33000, 500])
    c = Case(gpu_device, F32, B=1, Nq=34000, Nk=130, H=1, D=8, segments=(seg, torch.tensor([[0] * 40 + [1] * 40 + [2] * 45 + [-1] * 5])))
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,H,Hk", [(8, 8, 2), (1, 32, 1), (11, 3, 1), (1, 33, 1), (17, 4, 2)])
def test_rows_about_one_operand(gpu_device, dtype, Nq, H, Hk):
    """31 to 34 (query, head) rows over a key head, about the 32 that the cache kernel takes; keys of several
    workgroups, packed and not."""
    c = Case(gpu_device, dtype, B=2, Nq=Nq, Nk=2100, H=H, Hk=Hk, D=64, causal=True, lengths=[2100, 1025], radius=16)
    check([c.call().detach()], c.exact(train=False))
    c = Case(gpu_device, dtype, B=2, Nq=Nq, Nk=2100, H=H, Hk=Hk, D=64,
             segments=(torch.full((2, Nq), 1), packed(2, 2100, [300, 1400, 200], hole=9)))
    check([c.call().detach()], c.exact(train=False))
    check(c.step(), c.exact())


def test_rows_far_apart_in_memory(gpu_device):
    """Rows of a cache 2^16 values apart, so that the last lie beyond 2^32 bytes; and the widest stride there is."""
    room = torch.empty(36000 << 16, dtype=BF16, device=gpu_device)
    for rows, stride, Nq in ((36000, 1 << 16, 1), (36000, 1 << 16, 60), (270, 1 << 23, 40)):
        c = Case(gpu_device, BF16, B=1, Nq=Nq, Nk=rows, H=1, D=64, causal=True)
        far = room[:rows * stride].view(1, rows, 1, stride)
        far[..., :64] = c.k
        far[..., 64:128] = c.v
        want = c.step()
        c.k, c.v = far[..., :64], far[..., 64:128]
        got = c.step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_single_row_of_any_stride(gpu_device):
    """The stride of a dimension of one row says nothing: none, or a huge one."""
    c = Case(gpu_device, BF16, B=2, Nq=1, H=2, D=32)
    want = c.step()
    q, k, v = (t.detach() for t in (c.q, c.k, c.v))
    for stride in (0, 8, 1 << 40):
        c.q, c.k, c.v = (t.as_strided(t.shape, (64, stride, 32, 1)) for t in (q, k, v))
        assert all(torch.equal(a, b) for a, b in zip(c.step(), want))


def test_scores_far_apart(gpu_device):
    """Scores of hundreds: the running maximum moves many times and nothing overflows."""
    c = Case(gpu_device, BF16, B=1, Nq=300, H=2, D=64, spread=6.0)
    check(c.step(), c.exact())
    c = Case(gpu_device, F32, B=1, Nq=300, H=2, D=64, spread=6.0, causal=True)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(gpu_device, dtype):
    base = Case(gpu_device, dtype, B=2, Nq=90, H=4, Hk=4, D=24, causal=True)
    want = base.step()
    qkv = torch.stack([base.q.detach(), base.k.detach(), base.v.detach()], 2)   # [B, N, 3, H, D]
    odd = torch.zeros(qkv.numel() + 1, dtype=dtype, device=gpu_device)
    odd[1:] = qkv.flatten()
    for src in (qkv, odd[1:].view(qkv.shape)):       # projections side by side, as they come; rows off 16 bytes: copied
        base.q, base.k, base.v = (src[:, :, t].detach() for t in range(3))
        assert all(torch.equal(a, b) for a, b in zip(base.step(), want))
    base.q, base.k, base.v = (t.detach().transpose(1, 2).contiguous().transpose(1, 2) for t in (base.q, base.k, base.v))
    base.do = base.do.transpose(1, 2).contiguous().transpose(1, 2)
    assert all(torch.equal(a, b) for a, b in zip(base.step(), want))
    base.do = torch.ones_like(base.do[:, :1, :1, :1]).expand(2, 90, 4, 24)
    check(base.step(), base.exact())


def test_broadcast_keys_and_heads(gpu_device):
    """Keys shared by a batch or by heads through expand: gradients are summed onto the one copy."""
    c = Case(gpu_device, F32, B=3, Nq=60, H=4, D=32)
    k, v = (t[:1, :, :1].detach().requires_grad_(True) for t in (c.k, c.v))
    c.k, c.v = k.expand(3, 60, 4, 32), v.expand(3, 60, 4, 32)
    o = attention(c.q, c.k, c.v)
    gk, gv = torch.autograd.grad(o, (k, v), c.do)
    want = c.exact()
    for g, (value, bound) in ((gk, want[2]), (gv, want[3])):
        assert bool(((g.double() - value.sum((0, 2), keepdim=True)).abs() <= bound.sum((0, 2), keepdim=True) + 12 * U * value.abs().sum((0, 2), keepdim=True)).all())


def test_fp32_under_autocast_and_mixed_table(gpu_device):
    c = Case(gpu_device, F32, B=1, Nq=80, H=2, D=32, radius=9)
    with torch.autocast("cuda", dtype=BF16):
        got = c.call()
    assert got.dtype == F32
    low = Case(gpu_device, BF16, B=1, Nq=80, H=2, D=32, radius=9, tdtype=F32)
    assert torch.equal(got, low.call().float())
    check(low.step(), low.exact())


def test_prefix_without_a_causal_mask_changes_nothing(gpu_device):
    c = Case(gpu_device, BF16, B=2, Nq=80, H=2, D=32)
    want = c.call()
    assert torch.equal(c.call(prefix=torch.tensor([7, 0], device=gpu_device)), want)


@pytest.mark.parametrize("kw", [dict(B=1, Nq=400, H=2, D=64, radius=64, segments=packed(1, 400, [150, 200])),
                                dict(B=2, Nq=1, Nk=3000, H=8, Hk=2, D=64, causal=True, lengths=[3000, 1200])],
                         ids=["packed", "token"])
def test_same_bits_other_stream_and_replays(gpu_device, kw):
    c = Case(gpu_device, BF16, **kw)
    want = c.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = c.step()
    for r in range(4):
        with torch.no_grad():
            c.q.mul_(-0.75)
            if c.lengths is not None:
                c.lengths.sub_(11)
        graph.replay()
        want = c.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), r


def test_two_graphs_do_not_share_space(gpu_device):
    a = Case(gpu_device, BF16, B=1, Nq=1, Nk=3000, H=8, Hk=2, D=64, causal=True)
    b = Case(gpu_device, BF16, B=1, Nq=1, Nk=2000, H=8, Hk=2, D=64, causal=True, seed=1)
    want = a.call(), b.call()
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.call())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_dispatcher_route(gpu_device):
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    c = Case(gpu_device, BF16, B=1, Nq=90, H=2, D=32, radius=5, causal=True)
    want = c.step()
    with Look():
        got = c.step()
    assert any("bioemu_mi355x.attention" in s for s in seen) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradient_against_differences(gpu_device):
    """Central differences of f = sum(o do) along random directions: off by h^2/6 of the third derivative and
    2 * 2^-24 * sum|o do| / h; with h = 2^-5 and scores of order 1 both are below 2^-7 of the sizes compared."""
    c = Case(gpu_device, F32, B=1, Nq=24, H=2, D=16, radius=4, cap=3.0, causal=True)
    got = c.step()
    h = 2.0 ** -5
    for leaf, grad in zip((c.q, c.k, c.v, c.table), got[1:]):
        v = torch.randn_like(leaf)
        with torch.no_grad():
            keep = leaf.clone()
            leaf.copy_(keep + h * v)
            up = (c.call().double() * c.do.double()).sum()
            leaf.copy_(keep - h * v)
            down = (c.call().double() * c.do.double()).sum()
            leaf.copy_(keep)
        assert abs((up - down) / (2 * h) - (grad.double() * v.double()).sum()) <= 2.0 ** -7 * (grad * v).abs().double().sum() + 1e-3


def test_norm_relative_positions_and_attention_together(gpu_device):
    """A packed training step through the three operators and library products, against the same step in float64
    (plain torch).  fp32: each operator is within 1e-5 of its own sizes; four of them in a row, 1e-4 of the largest
    gradient."""
    torch.manual_seed(0)
    N, C, H = 120, 64, 4
    norm, att = LayerNorm(C).to(gpu_device), SequenceAttention(H, radius=8).to(gpu_device)
    rel = RelativePosition(H, radius=8).to(gpu_device)
    with torch.no_grad():
        att.bias.normal_()
        norm.weight.add_(0.1 * torch.randn_like(norm.weight))
    w = torch.nn.Linear(C, 3 * C, bias=False).to(gpu_device)
    x = torch.randn(1, N, C, device=gpu_device, requires_grad=True)
    seg = packed(1, N, [50, 60]).to(gpu_device)
    pos = torch.arange(N, device=gpu_device)[None]
    params = [x, norm.weight, norm.bias, w.weight, att.bias, rel.weight]

    def own():
        q, k, v = w(norm(x)).view(1, N, 3, H, C // H).unbind(2)
        return (att(q, k, v, segments=seg) ** 2).sum() + (rel(pos, seg.clamp(min=0)) ** 2).mean()

    def plain(ps):
        x, nw, nb, w, bias, rw = ps
        y = torch.nn.functional.layer_norm(x, (C,), nw, nb, norm.eps) @ w.t()
        q, k, v = (t.transpose(1, 2) for t in y.view(1, N, 3, H, C // H).unbind(2))
        off = (pos[:, None, :] - pos[:, :, None]).clamp(-8, 8) + 8
        s = torch.matmul(q, k.transpose(2, 3)) * (C // H) ** -0.5 + bias[off].permute(0, 3, 1, 2)
        ok = ((seg[:, :, None] == seg[:, None]) & (seg >= 0)[:, :, None])[:, None]
        p = torch.where(ok.any(-1, keepdim=True), s.masked_fill(~ok, -1e30).softmax(-1), 0.0)
        o = torch.matmul(torch.where(ok, p, 0.0), v)
        ch = seg.clamp(min=0)
        e = rw[torch.where(ch[:, None] == ch[:, :, None], off, rw.shape[0] - 1)]
        return (o ** 2).sum() + (e ** 2).mean()

    got = torch.autograd.grad(own(), params)
    exact = [p.detach().double().requires_grad_(True) for p in params]
    want = torch.autograd.grad(plain(exact), exact)
    for g, t in zip(got, want):
        assert (g.double() - t).abs().max() <= 1e-4 * t.abs().max()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_then_tokens_as_one_pass(gpu_device, dtype):
    """Serving: a prompt of 150 rows, then eleven single tokens and a pair against the growing cache (room for 300, NaN
    behind what is written), within the bounds of the one causal pass over all of them."""
    B, N, H, Hk, D = 2, 163, 8, 2, 64
    c = Case(gpu_device, dtype, B=B, Nq=N, H=H, Hk=Hk, D=D, causal=True, radius=30, num_buckets=32)
    (value, bound), = c.exact(train=False)
    cache = torch.full((2, B, 300, Hk, D), math.nan, dtype=dtype, device=gpu_device)
    at = 0
    for n in (150, *([1] * 11), 2):
        cache[0, :, at:at + n], cache[1, :, at:at + n] = c.k[:, at:at + n], c.v[:, at:at + n]
        o = attention(c.q[:, at:at + n], cache[0], cache[1], causal=True, bias_table=c.table, bias_buckets=c.buckets,
                      cache_lengths=torch.full((B,), at + n, device=gpu_device))
        check([o], [(value[:, at:at + n], bound[:, at:at + n])])
        at += n
    assert at == N


def test_two_threads_at_once(gpu_device):
    """Two threads train on streams of their own; every step gives the bits of the same step alone."""
    import threading

    cases = [Case(gpu_device, BF16, B=1, Nq=300, H=2, D=64, radius=16, segments=packed(1, 300, [100, 150])),
             Case(gpu_device, F32, B=2, Nq=1, Nk=2500, H=8, Hk=2, D=32, causal=True)]
    want = [c.step() for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(c, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = c.step()
                torch.cuda.current_stream().synchronize()
                wrong.extend(n for n, (g, t) in enumerate(zip(got, w)) if not torch.equal(g, t))

    threads = [threading.Thread(target=work, args=p) for p in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_gradients_of_some_inputs_only(gpu_device):
    c = Case(gpu_device, BF16, B=1, Nq=130, H=4, Hk=2, D=32, radius=8, causal=True)
    want = c.step()
    leaves = (c.q, c.k, c.v, c.table)
    for on in ((0,), (1, 2), (3,)):
        for n, t in enumerate(leaves):
            t.requires_grad_(n in on)
        got = torch.autograd.grad(c.call(), [leaves[n] for n in on], c.do)
        assert all(torch.equal(g, want[1 + n]) for g, n in zip(got, on))


@pytest.mark.parametrize("seed", range(40))
def test_arguments_in_any_combination(gpu_device, seed):
    """Sizes, types, head layouts, masks, lengths, bias and cap drawn together."""
    import random

    r = random.Random(seed)
    B, Hk, D = r.randint(1, 3), r.randint(1, 3), r.choice([8, 16, 24, 32, 40, 64, 72, 96, 128])
    H, Nq, Nk = Hk * r.randint(1, 4), r.choice([1, 2, 7, 31, 33, 64, 100, 129, 200, 257]), r.choice([1, 5, 32, 63, 65, 130, 255, 400, 700])
    kw = {}
    if r.random() < 0.5:
        kw["causal"] = True
        if r.random() < 0.5:
            kw["prefix"] = [r.randint(-1, Nk + 3) for _ in range(B)]
    if r.random() < 0.5:
        kw["lengths"] = [r.choice([0, 1, Nk, Nk + 9, r.randint(0, Nk)]) for _ in range(B)]
    if r.random() < 0.5:
        ids = [-1, *range(r.randint(1, 4))]
        order = sorted if r.random() < 0.5 else list
        kw["segments"] = tuple(torch.tensor([order(r.choices(ids, k=n)) for _ in range(B)]) for n in (Nq, Nk))
    if r.random() < 0.6:
        radius = r.choice([0, 1, 9, 64, 200])
        kw |= dict(radius=radius, num_buckets=None if radius < 120 else 32, tdtype=r.choice([None, F32, BF16]))
    if r.random() < 0.4:
        kw["cap"] = r.choice([0.5, 3.0, 40.0])
    c = Case(gpu_device, r.choice([BF16, F32]), B=B, Nq=Nq, Nk=Nk, H=H, Hk=Hk, D=D, seed=seed,
             scale=r.choice([None, None, 0.3, -0.2]), spread=r.choice([1.0, 3.0]), **kw)
    print(seed, c.q.dtype, B, Nq, Nk, H, Hk, D, {k: v for k, v in kw.items() if k != "segments"}, flush=True)
    check([c.call().detach()], c.exact(train=False))
    check(c.step(), c.exact())


def test_fake_tensors(gpu_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        c = [torch.empty(2, 30, h, 32, device="cuda", dtype=BF16, requires_grad=True) for h in (4, 2, 2)]
        table = torch.empty(9, 4, device="cuda", requires_grad=True)
        o = attention(*c, bias_table=table, bias_buckets=torch.empty(9, dtype=torch.uint8, device="cuda"))
        g = torch.autograd.grad(o, c + [table], torch.empty_like(o))
        assert o.shape == c[0].shape and [t.shape for t in g] == [t.shape for t in c + [table]]


def test_zero_sizes(gpu_device):
    c = Case(gpu_device, F32, B=2, Nq=5, Nk=0, H=2, D=16, radius=2)
    got = c.step()
    assert bool((got[0] == 0).all()) and bool((got[1] == 0).all()) and got[2].shape == (2, 0, 2, 16)
    assert bool((got[4] == 0).all())
    for shape in ((0, 5), (2, 0)):
        q = torch.randn(*shape, 2, 16, device=gpu_device, requires_grad=True)
        k = torch.randn(shape[0], 7, 2, 16, device=gpu_device, requires_grad=True)
        o = attention(q, k, k)
        gq, gk = torch.autograd.grad(o.sum(), (q, k))
        assert o.shape == q.shape and gq.shape == q.shape and bool((gk == 0).all())


def test_refusals(gpu_device):
    c = Case(gpu_device, F32, B=2, Nq=12, H=4, Hk=2, D=16, radius=2)
    q, k, v = c.q, c.k, c.v
    seg = torch.zeros(2, 12, dtype=torch.int32, device=gpu_device)
    one = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    bad = [
        (dict(q=q.half()), "fp32 or bf16"), (dict(q=q.bfloat16()), "q is"), (dict(q=q[0]), "must be"),
        (dict(v=v[:, :5]), "attention: q"), (dict(q=q[:, :, :3]), "heads over"), (dict(k=k.cpu(), v=v.cpu()), "on cpu"),
        (dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), "multiple of 8"),
        (dict(q=torch.zeros(1, 2, 1, 136, device=gpu_device), k=torch.zeros(1, 2, 1, 136, device=gpu_device),
              v=torch.zeros(1, 2, 1, 136, device=gpu_device)), "multiple of 8"),
        (dict(segments=seg[:, :5]), "shape"), (dict(segments=seg.float()), "whole numbers"),
        (dict(key_segments=seg), "come together"),
        (dict(prefix=one[:1], causal=True), "shape"), (dict(cache_lengths=one[:1]), "shape"), (dict(cap=0.0), "cap"),
        (dict(cap=float("inf")), "cap"), (dict(cap=1e6), "cap"), (dict(cap=1e-60), "cap"), (dict(cap=1e-35), "cap"), (dict(scale=float("nan")), "scale"),
        (dict(bias_table=c.table), "buckets"), (dict(bias_buckets=c.buckets), "buckets"),
        (dict(bias_table=c.table, bias_buckets=c.buckets[:-1]), "radius"),
        (dict(bias_table=c.table[:, :3], bias_buckets=c.buckets), "shape"),
        (dict(bias_table=c.table, bias_buckets=torch.zeros(1027, dtype=torch.uint8, device=gpu_device)), "at most 512"),
        (dict(bias_table=torch.zeros(257, 4, device=gpu_device), bias_buckets=c.buckets), "at most 256"),
    ]
    for kw, what in bad:
        args = dict(q=q, k=k, v=v) | kw
        with pytest.raises(ValueError, match=what):
            attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)


LONG = [(F32, 34000), (BF16, 65600)]   # just past 1024 blocks of 32 and of 64 rows


@pytest.mark.parametrize("dtype,Nk", LONG)
@pytest.mark.parametrize("kw", [dict(), dict(causal=True)], ids=["plain", "causal"])
def test_log_sums_past_1024_blocks_of_keys(gpu_device, dtype, Nk, kw):
    """Without segments every key counts once in the saved log-sum too, which dk and dv are made from.  A log-sum is off
    by a score's error e, by n u, the adds of n weights, and by 4 u of its two parts, each below 64."""
    c = Case(gpu_device, dtype, B=1, Nq=130, Nk=Nk, H=1, D=8, **kw)
    got, want = c.step(), c.exact()
    lse = torch_op("attention_train")(c.q.detach(), c.k.detach(), c.v.detach(), None, None, None, None, None, None,
                                      8 ** -0.5, 0.0, c.causal)[2].double().sum(0) * math.log(2)
    q, k = (t.detach().double().transpose(1, 2) for t in (c.q, c.k))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * 8 ** -0.5
    size = torch.matmul(q.abs(), k.abs().transpose(2, 3).contiguous()) * 8 ** -0.5
    exact = s.masked_fill(~c.allowed()[0][:, None], -math.inf).logsumexp(-1)
    off = (16 * U * size + 8 * U * s.abs()).amax(-1) + Nk * U + 4 * 64 * U
    assert bool(((lse - exact).abs() <= off).all()), (lse - exact).abs().max().item()
    check([got[n] for n in (0, 2, 3)], [want[n] for n in (0, 2, 3)], ("o", "dk", "dv"))


@pytest.mark.parametrize("dtype,Nk", LONG)
@pytest.mark.parametrize("Nq,kw", [(130, dict()), (130, dict(causal=True, radius=20)), (1, dict(radius=16)),
                                   (1, dict(causal=True, cap=4.0))], ids=["plain", "causal_bias", "token_bias", "token_capped"])
def test_gradients_past_1024_blocks_of_keys(gpu_device, dtype, Nk, Nq, kw):
    """Every key counts once in dq and in the table's gradient, after either form of the forward pass."""
    c = Case(gpu_device, dtype, B=1, Nq=Nq, Nk=Nk, H=1, D=8, **kw)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype,Nq", LONG)
@pytest.mark.parametrize("kw", [dict(), dict(causal=True, prefix=[50]), dict(cap=4.0, radius=20)],
                         ids=["plain", "prefix", "bias_capped"])
def test_gradients_past_1024_blocks_of_queries(gpu_device, dtype, Nq, kw):
    """Every query counts once in dk and dv."""
    c = Case(gpu_device, dtype, B=1, Nq=Nq, Nk=130, H=2, Hk=1, D=8, **kw)
    check(c.step(), c.exact())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_rows_that_see_nothing_hold_does_not_count(gpu_device, dtype):
    """A query of a segment that no key has, and one whose keys all have a bias of -infinity: whatever its gradient
    holds, it has none and gives none."""
    k_seg = packed(2, 150, [70, 75])
    q_seg = k_seg.clone()
    q_seg[:, 20:25] = q_seg[:, 90] = 7
    c = Case(gpu_device, dtype, B=2, Nq=150, H=2, D=64, segments=(q_seg, k_seg), radius=16)
    orphan = (q_seg == 7).to(gpu_device)
    want = c.step()
    for value in (math.nan, math.inf):
        c.do[orphan] = value
        c.q.data[orphan] = value
        got = c.step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(bool((t[orphan] == 0).all()) for t in got[:2])
    c = Case(gpu_device, dtype, B=1, Nq=60, H=2, D=32, radius=3)
    c.table[:, 1] = -math.inf
    want = c.step()
    c.do[:, :, 1] = math.nan
    got = c.step()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((got[1][:, :, 1] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("cap", [30.0, 4096.0, 4097.0, 1e5])
@pytest.mark.parametrize("Nq", [1, 70])
def test_capped_scores_themselves(gpu_device, dtype, D, cap, Nq):
    """Every query sees one key, so its log-sum is its score and its weight is 1 in both directions.  A score is off by
    (D + 8) u of its product and 16 u of itself (scale, cap, bias, log2 e, the tanh's few last places); up to a cap of
    4096 in bf16 by 4e-7 of the cap more."""
    n = torch.arange(Nq)[None]
    c = Case(gpu_device, dtype, B=1, Nq=Nq, H=2, D=D, segments=n, cap=cap, radius=2, spread=4.0)
    want = c.exact()
    lse = torch_op("attention_train")(c.q, c.k, c.v, c.table, c.buckets, c.segments, c.segments, None, None, D ** -0.5,
                                      cap, False)[2].double().sum(0) * math.log(2)
    q, k = (t.double().transpose(1, 2) for t in (c.q, c.k))
    x, size = (q * k).sum(-1) * D ** -0.5, (q * k).abs().sum(-1) * D ** -0.5
    bias = c.table.double()[2][None, :, None]
    s = cap * torch.tanh(x / cap)
    off = (D + 8) * U * size + 16 * U * (s.abs() + bias.abs()) + (4e-7 * cap if dtype == BF16 and cap <= 4096 else 0.0)
    err = (lse - s - bias).abs()
    print(f"off {err.max().item():.2e}, allowed {off.max().item():.2e}", flush=True)
    assert bool((err <= off).all())
    got = c.step()
    check(got, want)
    assert torch.equal(got[0], c.v.detach())
    # the backward pass takes its weight from a score summed in another order and the log-sum: 1 off by 2 off + 8 u, and
    # rounded as an operand and as the result
    off = (2 * off + 8 * U + 2 * _half(dtype)).transpose(1, 2)[..., None]
    assert bool(((got[3] - c.do).double().abs() <= off * c.do.double().abs()).all())
