"""Edges of rotary positions and the paged cache against float64: the table's end, numbers of 64 bits, caches that share
memory, workgroups of several sequences or of more values than their threads hold at once.  Bounds as derived in the
files of the operators' other tests."""

from __future__ import annotations

import pytest
import torch
from test_paged_cache_gpu import Case, _close, _turned
from test_rotary_gpu import check, exact, rand

from bioemu2_amd.paged_cache import paged_append
from bioemu2_amd.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


# ----------------------------------------------------------------------------
# More than the threads of a workgroup hold at once, and several sequences in one
# ----------------------------------------------------------------------------
MANY = [  # B, N, H, Hk, D, rot
    (1, 3, 64, 2, 128, 6),        # an odd number of pairs: pieces of one pair, 4224 of them a token
    (2, 1, 48, 8, 512, 512), (1, 2, 40, 24, 512, 20),
    (3, 1001, 3, 1, 24, 24),      # two tokens a workgroup: the sequences' borders inside one, the last of one token
    (3, 6667, 1, 1, 8, 4)]        # sixteen


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D,rot", MANY)
def test_rotary_by_workgroups(gpu_device, dtype, interleaved, B, N, H, Hk, D, rot):
    q, k = rand(B, N, H, D, dtype=dtype), rand(B, N, Hk, D, dtype=dtype, seed=1)
    pos = torch.randint(-5000, 5000, (B, N), generator=torch.Generator().manual_seed(N), dtype=I32).cuda()
    f = rotary_frequencies(rot, device="cuda")
    for at in (pos, None):
        y = rotary(q, k, at, f, interleaved=interleaved, magnitude=1.25)
        check(y[0], exact(q, at, f, interleaved, 1.25))
        check(y[1], exact(k, at, f, interleaved, 1.25))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D,rot", MANY)
def test_append_by_workgroups(gpu_device, dtype, interleaved, B, N, H, Hk, D, rot):
    page = 20
    counts = [N, N // 2, max(N - 3, 0)][:B]
    lengths = [N + 45, N // 2 + 7, N][:B]
    q, k, v = (rand(B, N, h, D, dtype=dtype, seed=s) for s, h in enumerate((H, Hk, Hk)))
    used = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(used) + 1, generator=torch.Generator().manual_seed(N))
    table = torch.full((B, max(used)), -1, dtype=I32)
    for b in range(B):
        table[b, :used[b]] = order[sum(used[:b]):sum(used[:b + 1])].to(I32)
    keys, values = (rand(sum(used) + 1, page, Hk, D, dtype=dtype, seed=s) for s in (3, 4))
    k0, v0 = keys.clone(), values.clone()
    f = rotary_frequencies(rot, device="cuda")
    got = paged_append(keys, values, k, v, table.cuda(), torch.tensor(lengths, dtype=I32, device="cuda"),
                       counts=torch.tensor(counts, dtype=I32, device="cuda"), q=q, frequencies=f, interleaved=interleaved,
                       magnitude=1.5)
    for b, n in enumerate(counts):
        pos = torch.arange(lengths[b] - n, lengths[b])
        at = (table[b][pos // page].long().cuda(), (pos % page).cuda())
        _close(got[b, :n], _turned(q[b, :n], pos.cuda(), f, interleaved, 1.5))
        _close(keys[at], _turned(k[b, :n], pos.cuda(), f, interleaved, 1.5))
        assert torch.equal(values[at], v[b, :n]) and bool((got[b, n:] == 0).all())
        keys[at], values[at] = k0[at], v0[at]
    assert torch.equal(keys, k0) and torch.equal(values, v0)     # nothing else was written


# ----------------------------------------------------------------------------
# Sequences longer than their table
# ----------------------------------------------------------------------------
def _past_the_table(c, width):
    return [torch.arange(k.shape[0], device="cuda") >= width * c.page for k, _ in c.dense]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Nq", [1, 4, 40])
@pytest.mark.parametrize("width", [6, 80])
def test_positions_past_the_table(gpu_device, dtype, causal, Nq, width):
    """Queries keep the positions that the lengths give them; only the keys end with the table."""
    room = 16 * width
    lengths = [room + 4, room, room + 30, 20, room + 1000]
    c = Case(lengths, dtype, Nq=Nq, width=width, radius=8, causal=causal, counts=[min(Nq, 8), Nq, Nq, min(Nq, 20), Nq])
    c.check(hidden=_past_the_table(c, width))


def test_lengths_at_the_end_of_32_bits(gpu_device):
    c = Case([64, 64], Nq=3, page=16, radius=8, counts=[3, 1])
    c.lengths.fill_(2 ** 31 - 1)
    far = c.call()
    c.lengths.fill_(2 ** 20)
    assert torch.equal(far, c.call())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_then_attend_across_the_tables_end(gpu_device, dtype):
    """Eight new rows of which four have a slot: each row sees what was written up to its own position."""
    c = Case([100, 60], dtype, Nq=8, width=6, radius=8)
    keys, values = c.keys.clone(), c.values.clone()
    k, v = (torch.stack([s[n][-8:] for s in c.dense]) for n in (0, 1))
    for b, n in enumerate((100, 60)):
        at = torch.arange(n - 8, min(n, 96), device="cuda")
        c.keys[c.table[b, at // 16].long(), at % 16] = c.values[c.table[b, at // 16].long(), at % 16] = 0
    paged_append(c.keys, c.values, k, v, c.table, c.lengths)
    for got, want in ((c.keys, keys), (c.values, values)):
        for b, n in enumerate((96, 60)):
            at = torch.arange(n, device="cuda")
            where = c.table[b, at // 16].long(), at % 16
            assert torch.equal(got[where], want[where])
    c.check(hidden=_past_the_table(c, 6))


# ----------------------------------------------------------------------------
# Numbers of 64 bits
# ----------------------------------------------------------------------------
def test_tables_and_lengths_of_64_bits(gpu_device):
    """What 32 bits do not hold names no page, is past any table, or below every length."""
    c = Case([64, 100, 32], page=16)
    table, lengths = c.table.long(), c.lengths.long()
    table[0, 1], table[1, 0], table[2, 0] = 2 ** 32, 2 ** 33 + 1, -2 ** 32
    c.table[0, 1] = c.table[1, 0] = c.table[2, 0] = -1
    lengths[1] += 2 ** 32
    c.lengths[1] = 2 ** 31 - 1
    counts = torch.tensor([1, 2 ** 32 + 1, -2 ** 40], device="cuda")
    c.counts = torch.tensor([1, 1, 0], dtype=I32, device="cuda")
    want = c.call()
    c.table, c.lengths, c.counts, want_of = table, lengths, counts, (c.table, c.lengths, c.counts)
    # as bits: with its length past the table, sequence 1 sees slots that hold NaN
    assert torch.equal(c.call().view(torch.int16), want.view(torch.int16)) and want[0].isfinite().all()
    k = torch.ones(3, 1, 2, 32, dtype=BF16, device="cuda")
    stores = [(c.keys.clone(), c.values.clone()) for _ in range(2)]
    for (keys, values), (t, n, m) in zip(stores, ((table, lengths, counts), want_of)):
        t = t.clone()
        t[0, 3] = t[0, 1]      # the new token's page: none
        paged_append(keys, values, k, k, t, n, counts=m)
    for got, want in zip(*stores):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    assert torch.equal(stores[0][0].view(torch.int16), c.keys.view(torch.int16))     # nothing was written


# ----------------------------------------------------------------------------
# Caches that share memory
# ----------------------------------------------------------------------------
def _append_ones(keys, values):
    """Every slot of every page gets keys 1 and values 2."""
    pages, page = keys.shape[:2]
    k = torch.ones(1, pages * page, *keys.shape[2:], dtype=keys.dtype, device="cuda")
    paged_append(keys, values, k, 2 * k, torch.arange(pages, dtype=I32, device="cuda")[None],
                 torch.tensor([pages * page], dtype=I32, device="cuda"))


def test_parts_of_one_allocation(gpu_device):
    P, S, H, D = 3, 4, 2, 16
    for whole, dim in [((2, P, S, H, D), 0), ((P, 2, S, H, D), 1), ((P, S, 2, H, D), 2), ((P, S, H, 2, D), 3),
                       ((P, H, 2, S, D), 2)]:
        both = torch.zeros(whole, dtype=BF16, device="cuda")
        keys, values = both.select(dim, 0), both.select(dim, 1)
        if whole[1] == H:
            keys, values = keys.transpose(1, 2), values.transpose(1, 2)
        _append_ones(keys, values)
        assert bool((keys == 1).all()) and bool((values == 2).all())
        _append_ones(values, keys)
        assert bool((keys == 2).all()) and bool((values == 1).all())


def test_slots_in_the_same_place_are_refused(gpu_device):
    both = torch.zeros(6, 4, 2, 16, dtype=F32, device="cuda")
    flat = both.flatten()
    same = lambda *st, at=0: flat.as_strided((2, 4, 2, 16), (*st, 1), at)  # noqa: E731
    for keys, values in [(both, both), (both[:4], both[2:]), (both[:, :3], both[:, 1:]), (both[..., :8], both[..., 4:12]),
                         (both[:3], both[2:5]),
                         (same(128, 32, 16), same(128, 16, 64, at=64)), (same(64, 32, 16), both[4:]),
                         (same(16, 32, 16), both[2:4]), (same(128, 0, 16), both[2:4]), (both[4:], same(128, 8, 64))]:
        with pytest.raises(ValueError):
            _append_ones(keys, values)
    assert both.abs().max() == 0


def test_any_layout_within_one_allocation(gpu_device):
    """Against the sets of places: what overlaps is refused; what does not is taken where steps are alike and each
    dimension steps over what lies within it."""
    import random

    r = random.Random(2)
    flat = torch.zeros(4096, dtype=BF16, device="cuda")
    size = []

    def layout():
        within, steps = 8, [0, 0, 0, 1]
        for d in r.sample(range(3), 3):
            steps[d] = within + 8 * r.choice([0, 0, 1, 3, 9]) - (8 if r.random() < 0.1 and within > 8 else 0)
            within += (size[d] - 1) * steps[d]
        return steps

    def steps_over(steps):
        within = 8
        for s, n in sorted((s, n) for s, n in zip(steps[:3], size[:3]) if n > 1):
            if s < within:
                return False
            within += (n - 1) * s
        return True

    taken = refused = 0
    while taken < 60 or refused < 60:
        size[:] = [r.randint(1, 3) for _ in range(3)] + [8]
        steps = [layout(), layout()]
        if r.random() < 0.8:
            steps[1] = steps[0]
        at = [8 * r.randint(0, 40) for _ in "kv"]
        places = [[a + i * st[0] + j * st[1] + k * st[2] + e for i in range(size[0]) for j in range(size[1])
                   for k in range(size[2]) for e in range(8)] for st, a in zip(steps, at)]
        clear = all(len(set(p)) == len(p) for p in places) and not set(places[0]) & set(places[1])
        keys, values = (flat.as_strided(size, st, a) for st, a in zip(steps, at))
        flat.zero_()
        try:
            _append_ones(keys, values)
        except ValueError as e:
            assert "share memory" in str(e), e
            refused += 1
            apart = max(places[0]) < min(places[1]) or max(places[1]) < min(places[0])
            # without need only where steps differ, or where a dimension steps into another
            assert not clear or not all(map(steps_over, steps)) or (steps[0] != steps[1] and not apart)
        else:
            taken += 1
            assert clear and bool((keys == 1).all()) and bool((values == 2).all())


# ----------------------------------------------------------------------------
# Long calls
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("n", [2 ** 28 + 5, 2 ** 31 - 17])
def test_more_tokens_than_a_launch_has_threads_for(gpu_device, n):
    """2^28 tokens and some, sixteen a workgroup of 256 threads, would be 2^32 threads; and the most that a call takes."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 34 * n + 2 ** 33:
        pytest.skip("not enough free memory")
    q = torch.empty(1, n, 1, 8, dtype=BF16, device="cuda").normal_()
    f = rotary_frequencies(4, device="cuda")
    got = rotary(q, None, None, f)[0]
    g = torch.Generator(device="cuda").manual_seed(0)
    some = torch.cat((torch.arange(2000, device="cuda"), torch.arange(n - 2000, n, device="cuda"),
                      torch.randint(0, n, (1000000,), generator=g, device="cuda")))
    check(got[:, some], exact(q[:, some], some.to(I32)[None], f))
    for at in range(0, n, 2 ** 27):                             # all rows: what does not turn
        assert torch.equal(got[0, at:at + 2 ** 27, 0, 4:], q[0, at:at + 2 ** 27, 0, 4:])
    del q, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths,heads", [([131072, 118528], 32), ([131072, 115680, 47936, 50784], 16)])
def test_parts_of_long_contexts(gpu_device, dtype, lengths, heads):
    Case(lengths, dtype, H=heads, Hk=heads, D=8, page=64).check()
