"""The relative-position embedding and its table's gradient against float64.

Forward: table values are exact, one fp32 add (2^-24 of the sum) and one rounding to the result's type (half a step).
Gradient: products with 0 and 1 are exact (an fp32 gradient goes in as three bf16 parts that hold its 24 bits), so only
adds are rounded.  A wave adds at most n = units / (8 workgroups) * 64 values of a bucket one after the other in the
worst case, 8 waves and then the workgroups follow: the error is at most (pairs per wave + 8 + groups / 64 + 8) 2^-24
times the sum of sizes.  The tests below bound pairs per wave by 64 ceil(units / (8 groups)), three parts each in fp32.
"""

from __future__ import annotations

import math

import pytest
import torch

from bioemu2_amd import _lib
from bioemu2_amd.relative_position import RelativePosition, distance_buckets, relative_position

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _half(dtype):
    return 2.0 ** -24 if dtype == F32 else torch.finfo(dtype).eps / 2


def _inputs(device, B, N, C, dtype, radius=32, num_buckets=None, chains=3, seed=0, add=True, tdtype=F32):
    g = torch.Generator().manual_seed(seed)
    buckets = distance_buckets(radius, num_buckets, device=device)
    nb = int(buckets.max()) + 2
    pos = (1 + 9 * (torch.rand(B, N, generator=g) < 0.05).int()).cumsum(1).int().to(device)
    ch = torch.randint(0, chains, (B, N), generator=g).int().to(device) if chains else None
    table = torch.randn(nb, C, generator=g).to(tdtype).to(device).requires_grad_(True)
    z = torch.randn(B, N, N, C, generator=g).to(dtype).to(device) if add else None
    return table, buckets, pos, ch, z, torch.randn(B, N, N, C, generator=g).to(dtype).to(device)


def _which(table, buckets, pos, ch):
    R = buckets.numel() // 2
    t = buckets.long()[(pos.long()[:, None, :] - pos.long()[:, :, None]).clamp(-R, R) + R]
    t = t.clamp(max=table.shape[0] - 1)
    return t if ch is None else torch.where(ch[:, None, :] == ch[:, :, None], t, table.shape[0] - 1)


def _check(table, buckets, pos, ch, z, dy, y, dt):
    t = _which(table, buckets, pos, ch)
    want = table.detach().double()[t]
    if z is not None:
        want = want + z.double()
    assert bool(((y.double() - want).abs() <= (_half(y.dtype) + 2 * U) * want.abs()).all())
    if dt is None:
        return
    B, N = pos.shape
    NB, C = table.shape
    flat, idx = dy.double().reshape(-1, C), t.reshape(-1)
    want = torch.zeros(NB, C, dtype=torch.float64, device=dy.device).index_add_(0, idx, flat)
    size = torch.zeros_like(want).index_add_(0, idx, flat.abs())
    units = B * N * math.ceil(N / 64)
    groups = _lib.lib().bioemu_relpos_bwd_workspace_bytes(B, N, C, NB) // (NB * C * 4)
    depth = (3 if dy.dtype == F32 else 1) * 64 * math.ceil(units / (8 * groups)) + 8 + groups / 64 + 8
    assert bool(((dt.double() - want).abs() <= depth * U * size + _half(dt.dtype) * want.abs()).all())


def _step(table, buckets, pos, ch, z, dy):
    y = relative_position(table, buckets, pos, ch, z=z, dtype=dy.dtype)
    return y.detach(), torch.autograd.grad(y, table, dy)[0]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,N,C,radius,nbk,chains", [
    (1, 1, 128, 32, None, 1), (2, 7, 16, 32, None, 0), (1, 64, 128, 32, None, 2), (1, 65, 64, 128, 64, 3),
    (3, 130, 128, 32, None, 1), (2, 97, 200, 64, 32, 2), (1, 50, 5, 3, None, 2), (1, 33, 1, 0, None, 2),
    (1, 70, 384, 127, None, 2), (1, 257, 16, 128, 252, 4), (2, 61, 33, 16, 4, 0)])
def test_step(gpu_device, dtype, B, N, C, radius, nbk, chains):
    args = _inputs(gpu_device, B, N, C, dtype, radius, nbk, chains, add=N % 2 == 0)
    _check(*args, *_step(*args))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_larger(gpu_device, dtype):
    args = _inputs(gpu_device, 1, 501, 128, dtype, seed=1)
    _check(*args, *_step(*args))


def test_bf16_table_and_unordered_positions(gpu_device):
    table, buckets, _, ch, z, dy = _inputs(gpu_device, 2, 90, 64, BF16, seed=2, tdtype=BF16)
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 90), device=gpu_device)   # differences beyond 32 bits
    y, dt = _step(table, buckets, pos, ch, z, dy)
    assert dt.dtype == BF16
    _check(table, buckets, pos, ch, z, dy, y, dt)


def test_map_values_past_the_table_count_as_the_last(gpu_device):
    table, buckets, pos, ch, z, dy = _inputs(gpu_device, 1, 40, 32, F32, seed=3)
    _check(table.detach()[:20].requires_grad_(True), buckets, pos, ch, z, dy,
           *_step(table.detach()[:20].requires_grad_(True), buckets, pos, ch, z, dy))


def test_gradient_of_z_and_strided_gradients(gpu_device):
    table, buckets, pos, ch, z, dy = _inputs(gpu_device, 1, 40, 32, F32, seed=4)
    z.requires_grad_(True)
    y = relative_position(table, buckets, pos, ch, z=z)
    gt, gz = torch.autograd.grad(y, (table, z), dy)
    assert torch.equal(gz, dy)
    y = relative_position(table, buckets, pos, ch, z=z.detach().transpose(1, 2))
    turned = dy.transpose(1, 2)
    gt2, = torch.autograd.grad(y, table, turned)
    _check(table, buckets, pos, ch, z.detach().transpose(1, 2), turned, y.detach(), gt2)
    y = relative_position(table, buckets, pos, ch)
    _check(table, buckets, pos, ch, None, torch.ones_like(dy), y.detach(), torch.autograd.grad(y.sum(), table)[0])


def test_gradient_against_differences(gpu_device):
    """The result is linear in the table: a difference over any h is the directional derivative, up to fp32 rounding of
    the results (2 * 2^-24 * size / h)."""
    table, buckets, pos, ch, _, dy = _inputs(gpu_device, 1, 30, 16, F32, seed=5, add=False)
    v = torch.randn_like(table)
    dt = _step(table, buckets, pos, ch, None, dy)[1]
    with torch.no_grad():
        a, b = (relative_position(table + s * v, buckets, pos, ch).double() for s in (0.5, -0.5))
    size = (a.abs() * dy.abs().double()).sum() + (b.abs() * dy.abs().double()).sum()
    assert abs(((a - b) * dy.double()).sum() - (dt.double() * v.double()).sum()) <= 4 * U * size + 1e-5 * (dt * v).abs().sum()


def test_same_bits_other_stream_and_replays(gpu_device):
    args = _inputs(gpu_device, 1, 300, 64, F32, seed=6)
    want = _step(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(*args)
    for k in range(4):
        args[5].mul_(-0.5)
        args[2].copy_(args[2].flip(1))
        graph.replay()
        want = _step(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), k


def test_module(gpu_device):
    mod = RelativePosition(32, radius=16).to(gpu_device)
    assert mod.num_buckets == 34 and set(mod.state_dict()) == {"weight"}
    pos = torch.arange(20, device=gpu_device)[None]
    out = mod(pos, torch.zeros_like(pos))
    assert out.shape == (1, 20, 20, 32) and torch.equal(out[0, 3, 5], mod.weight.detach()[18])
    out.square().sum().backward()
    assert torch.equal(mod.weight.grad[-1], torch.zeros(32, device=gpu_device))
    empty = mod(pos[:, :0])
    assert empty.shape == (1, 0, 0, 32)
    assert torch.equal(torch.autograd.grad(empty.sum(), mod.weight)[0], torch.zeros_like(mod.weight))


def test_refusals(gpu_device):
    table, buckets, pos, ch, z, _ = _inputs(gpu_device, 1, 12, 16, F32)
    big = torch.zeros(257, 16, device=gpu_device)
    for kw, what in ((dict(table=table.detach().half()), "fp32 or bf16"), (dict(buckets=buckets[:-1]), "radius"),
                     (dict(buckets=buckets.int()), "dtype"), (dict(positions=pos.float()), "whole numbers"),
                     (dict(positions=pos[0]), "positions"), (dict(chains=ch[:, :4]), "shape"),
                     (dict(z=z[..., :8]), "shape"), (dict(z=z, dtype=BF16), "dtype"), (dict(table=big), "at most 256"),
                     (dict(dtype=torch.float16), "fp32 or bf16"),
                     (dict(table=torch.zeros(4, 257, device=gpu_device)), "at most 256")):
        args = dict(table=table, buckets=buckets, positions=pos, chains=ch) | kw
        with pytest.raises(ValueError, match=what):
            relative_position(**args)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [1016, 1024, 1028, 1032, 2048, 2056, 4096])
def test_wide_rows(gpu_device, dtype, C):
    """Rows of more 16-byte pieces than a workgroup has threads, up to the limit; tables and z at any address."""
    if C % 8 and dtype == BF16:
        pytest.skip("not whole 16-byte pieces")
    args = _inputs(gpu_device, 2, 9, C, dtype, radius=3, chains=2, add=True)
    want = _step(*args)
    _check(*args, *want)
    table, buckets, pos, ch, z, dy = args
    odd = lambda t: torch.cat([t.new_zeros(1), t.detach().flatten()])[1:].view(t.shape)  # noqa: E731
    moved = (odd(table).requires_grad_(True), buckets, pos, ch, odd(z), odd(dy))
    assert moved[0].data_ptr() % 16 and moved[4].data_ptr() % 16
    assert all(torch.equal(a, b) for a, b in zip(_step(*moved), want))


def test_widths_past_the_limit(gpu_device):
    for C, dtype in ((4104, BF16), (4100, F32), (260, BF16)):
        table, buckets, pos, *_ = _inputs(gpu_device, 1, 4, C, dtype, radius=2, add=False)
        with pytest.raises(ValueError, match="at most"):
            relative_position(table, buckets, pos, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,C,radius", [(9, 16, 2), (70, 128, 32), (130, 33, 100)])
def test_gradients_that_are_not_finite_reach_their_own_bucket(gpu_device, dtype, N, C, radius):
    """Infinities, NaN and the type's largest values in some pairs: the sums of every other bucket and channel are as
    without them, within the bounds of any order of adds."""
    table, buckets, pos, ch, z, dy = _inputs(gpu_device, 2, N, C, dtype, radius, chains=2, add=False)
    pos = torch.arange(N, dtype=torch.int32, device=gpu_device).expand(2, N).contiguous()
    for i, j, channel, value in ((1, 3, 2, math.inf), (4, 4, C - 1, -math.inf), (5, 7, 0, math.nan),
                                 (8, 0, 5, torch.finfo(dtype).max), (2, 2, C - 1, math.inf)):
        dy[1, i, j, channel] = value
    _, dt = _step(table, buckets, pos, ch, None, dy)
    t = _which(table, buckets, pos, ch).reshape(-1)
    flat = dy.double().reshape(-1, C)
    zeros = torch.zeros(table.shape, dtype=torch.float64, device=gpu_device)
    want, size = zeros.index_add(0, t, flat), zeros.index_add(0, t, flat.abs())
    special = ~(want.abs() <= 1e38)
    assert 3 <= int(special.sum()) <= 5
    assert bool(((dt.double() - want).abs() <= 2 * N * N * 3 * U * size)[~special].all())
    assert bool(torch.equal(dt.double()[special].nan_to_num(0.5, 1.0, -1.0).sign(),
                            want[special].nan_to_num(0.5, 1.0, -1.0).sign()))
    assert bool((dt.isnan() == want.isnan()).all())
