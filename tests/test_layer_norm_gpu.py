"""LayerNorm and its gradients against float64.

Tolerances.  u = 2^-24 is half an fp32 step relative to a value.  A lane adds at most E values one after the other and a
row's lanes in at most 8 + 4 steps, so a sum of c terms is off by at most K u times the sum of their sizes, K = E + 12
(E <= 64).  With that, to first order (12 covers the handful of roundings of each product and of 1 / sqrt):
  d(xh) = u (K r max|x| + (K + 12) |xh|)
  d(y)  = |w| d(xh) + 2 u (|y| + |b|)
  d(dx) = r [u (K + 12) (|gy| + mean|gy| + |xh| mean|gy xh|) + d(xh) |mean gy xh| + |xh| mean(|gy| d(xh))]
          + 12 u |dx| + |dx| 2 d(r)/r, the last inside (K + 12)
  d(dw) = (D + 2) u sum|dy xh| + sum |dy| d(xh),  d(db) = D u sum|dy|
where D = rows / 1024 + 64 adds follow each other in a weight gradient.  A result in bf16 is off by half a step
more, 2^-8 of its value.
"""

from __future__ import annotations

import pytest
import torch

from bioemu2_amd import _lib
from bioemu2_amd.layer_norm import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 64 + 12
EPS = 1e-5
BF16, F32 = torch.bfloat16, torch.float32


def _half(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def _within(got, want, tol, what):
    got = got.double()
    over = (got - want).abs() - tol
    assert bool((over <= 0).all()), f"{what}: off by {(got - want).abs().max().item():.3e}, {int((over > 0).sum())} over"


def _check(x, w, b, dy, outs, eps=EPS):
    y, dx, dw, db = outs
    xd, dyd = x.detach().double(), dy.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    bd = torch.zeros_like(wd) if b is None else b.detach().double()
    mu = xd.mean(-1, keepdim=True)
    r = 1 / ((xd - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (xd - mu) * r
    gy = dyd * wd
    mg, mgx = gy.mean(-1, keepdim=True), (gy * xh).mean(-1, keepdim=True)
    dxh = U * (K * r * xd.abs().amax(-1, keepdim=True) + (K + 12) * xh.abs())
    want = xh * wd + bd
    _within(y, want, dxh * wd.abs() + 2 * U * (want.abs() + bd.abs()) + _half(y.dtype) * want.abs(), "y")
    if dx is not None:
        want = r * (gy - mg - xh * mgx)
        tol = r * (U * (K + 12) * (gy.abs() + gy.abs().mean(-1, keepdim=True) + xh.abs() * (gy * xh).abs().mean(-1, keepdim=True))
                   + dxh * mgx.abs() + xh.abs() * (gy.abs() * dxh).mean(-1, keepdim=True)) + (K + 24) * U * want.abs()
        # r itself is off by what the variance is: r^2 sum |x - mu| d(mu) / c, inside K r max|x|
        tol = tol + want.abs() * U * K * r * xd.abs().amax(-1, keepdim=True)
        _within(dx, want, tol + _half(dx.dtype) * want.abs(), "dx")
    depth = x.numel() // x.shape[-1] / 1024 + 64
    rows = tuple(range(x.ndim - 1))
    if dw is not None:
        want = (dyd * xh).sum(rows)
        _within(dw, want, (depth + 2) * U * (dyd * xh).abs().sum(rows) + (dyd.abs() * dxh).sum(rows)
                + _half(dw.dtype) * want.abs(), "dw")
    if db is not None:
        want = dyd.sum(rows)
        _within(db, want, depth * U * dyd.abs().sum(rows) + _half(db.dtype) * want.abs(), "db")


def _step(x, w, b, dy, eps=EPS):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = layer_norm(x, w, b, eps)
    g = iter(torch.autograd.grad(y, leaves, dy))
    return y.detach(), next(g), None if w is None else next(g), None if b is None else next(g)


def _inputs(device, rows, c, dtype, seed=0, wdtype=F32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) * 1.5 + torch.randn(c, generator=g)).to(dtype).to(device)
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(wdtype).to(device)
    b = (0.2 * torch.randn(c, generator=g)).to(wdtype).to(device)
    return x, w, b, torch.randn(rows, c, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 128), (3, 7), (513, 16), (300, 64), (77, 100), (4099, 128), (65, 256),
                                    (200, 333), (201, 384), (33, 512), (50, 768), (129, 1024), (9, 1030), (17, 2048),
                                    (5, 2999), (5, 4096), (3, 8192), (3, 16384)])
def test_layer_norm_step(gpu_device, dtype, rows, c):
    x, w, b, dy = _inputs(gpu_device, rows, c, dtype)
    _check(x, w, b, dy, _step(x, w, b, dy))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pair_representation(gpu_device, dtype):
    """Many rows: every workgroup walks, and the partial rows of all of them are added."""
    x, w, b, dy = _inputs(gpu_device, 301 * 301, 128, dtype, seed=1)
    shape = (1, 301, 301, 128)
    outs = _step(x.view(shape).detach(), w, b, dy.view(shape))
    assert outs[0].shape == shape and outs[1].shape == shape
    _check(x.view(shape), w, b, dy.view(shape), outs)


@pytest.mark.parametrize("w_on,b_on", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("wdtype", [BF16, F32])
def test_parameters_may_be_absent_or_bf16(gpu_device, w_on, b_on, wdtype):
    x, w, b, dy = _inputs(gpu_device, 70, 384, BF16, seed=2, wdtype=wdtype)
    w, b = (w if w_on else None), (b if b_on else None)
    outs = _step(x, w, b, dy)
    assert all(t is None or t.dtype == wdtype for t in outs[2:])
    _check(x, w, b, dy, outs)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("how", ["row_stride", "odd_stride", "offset", "transposed", "dy_expanded"])
def test_strides_and_alignment(gpu_device, dtype, how):
    x, w, b, dy = _inputs(gpu_device, 90, 200, dtype, seed=3)
    if how == "row_stride":
        x, w, b, dy = x[:, 8:136], w[:128].contiguous(), b[:128].contiguous(), dy[:, 64:192]
    elif how == "odd_stride":
        x, w, b, dy = x[:, 1:130], w[:129].contiguous(), b[:129].contiguous(), dy[:, 3:132]
    elif how == "offset":
        x = x.flatten()[1:1 + 89 * 200].view(89, 200)
        dy = dy[:89]
    elif how == "transposed":
        x, w, b, dy = x.t(), w[:90].contiguous(), b[:90].contiguous(), dy.t()
    else:
        dy = dy[:1].expand(90, 200)
    x = x.detach()
    _check(x, w, b, dy, _step(x, w, b, dy))


def test_large_mean_keeps_the_deviation(gpu_device):
    """Values near 1000 with deviations of 1: a second pass over the row, not E[x^2] - mean^2 (which would be off by
    1000^2 u K, 5 parts in 1000 of the variance)."""
    x, w, b, dy = _inputs(gpu_device, 64, 384, F32, seed=4)
    x = (x + 1000).detach()
    outs = _step(x, w, b, dy)
    _check(x, w, b, dy, outs)
    want = torch.nn.functional.layer_norm(x.detach().double(), (384,), w.detach().double(), b.detach().double(), EPS)
    # mean off by at most K u 1000 = 0.0045 deviations in the worst case; sums of random signs stay below a tenth of it
    assert (outs[0].double() - want).abs().max() < K * U * 1100 * 1.6


def test_not_finite_rows_stay_alone(gpu_device):
    x, w, b, dy = _inputs(gpu_device, 40, 128, F32, seed=5)
    want = _step(x.clone().detach(), w, b, dy)
    bad = x.detach().clone()
    bad[7, 3], bad[20, 100] = float("nan"), float("inf")
    got = _step(bad, w, b, dy)
    keep = [i for i in range(40) if i not in (7, 20)]
    for g, t in zip(got[:2], want[:2]):
        assert torch.equal(g[keep], t[keep]) and bool(g[[7, 20]].isnan().all())


def test_zero_rows_and_constant_rows(gpu_device):
    w = torch.ones(64, device=gpu_device, requires_grad=True)
    x = torch.empty(0, 64, device=gpu_device, requires_grad=True)
    y = layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    y = layer_norm(torch.full((3, 64), 7.0, device=gpu_device), w.detach(), None)
    assert torch.equal(y, torch.zeros_like(y))


def test_same_bits_every_time_and_on_another_stream(gpu_device):
    x, w, b, dy = _inputs(gpu_device, 30000, 128, BF16, seed=6)
    want = _step(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, t) for g, t in zip(got, want))


def test_captured_step_replays(gpu_device):
    x, w, b, dy = _inputs(gpu_device, 3000, 384, BF16, seed=7)
    for t in (x, w, b):
        t.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(x, w, b, dy)
    for k in range(4):
        with torch.no_grad():
            x.add_(0.25)
            dy.mul_(0.5)
        graph.replay()
        want = _step(x, w, b, dy)   # eager work between replays
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(outs, want)), k


def test_dispatcher_route_and_partial_gradients(gpu_device):
    """The registered op (a dispatch mode looks on) gives the direct call's bits; gradients nobody asks for are not made."""
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, w, b, dy = _inputs(gpu_device, 200, 384, F32, seed=8)
    want = _step(x, w, b, dy)
    with Look():
        got = _step(x, w, b, dy)
    assert any("layer_norm" in s for s in seen) and all(torch.equal(g, t) for g, t in zip(got, want))
    y = layer_norm(x.detach(), w.requires_grad_(True), b.detach())
    (dw,) = torch.autograd.grad(y, (w,), dy)
    assert torch.equal(dw, want[2])
    y = layer_norm(x.requires_grad_(True), w.detach(), None)
    (dx,) = torch.autograd.grad(y, (x,), dy)
    assert torch.equal(dx, want[1])


def test_module_matches_torch_state_dict_and_trains(gpu_device):
    mod = LayerNorm(96).to(gpu_device)
    mod.load_state_dict(torch.nn.LayerNorm(96).state_dict())
    x = torch.randn(5, 4, 96, device=gpu_device)
    mod(x).square().sum().backward()
    assert mod.weight.grad.shape == (96,) and bool(mod.weight.grad.isfinite().all())
    assert set(LayerNorm(8, bias=False).state_dict()) == {"weight"}


def test_gradient_against_differences(gpu_device):
    """(f(x + h v) - f(x - h v)) / 2h of a scalar f: off by h^2 |f'''| / 6 and 2 u |f| / h; h = 2^-6 keeps both below
    2^-9 of the directional derivative's size here (f is a sum of 12 * 64 values of order 1)."""
    x, w, b, dy = _inputs(gpu_device, 12, 64, F32, seed=9)
    outs = _step(x, w, b, dy)
    v = torch.randn(12, 64, device=gpu_device)
    h = 2.0 ** -6
    f = lambda t: (layer_norm(t, w.detach(), b.detach()).double() * dy.double()).sum()  # noqa: E731
    with torch.no_grad():
        fd = (f(x + h * v) - f(x - h * v)) / (2 * h)
    got = (outs[1].double() * v.double()).sum()
    assert abs(fd - got) <= 2.0 ** -9 * (outs[1].double() * v.double()).abs().sum()


def test_refusals(gpu_device):
    x = torch.randn(4, 64, device=gpu_device)
    w = torch.ones(64, device=gpu_device)
    for args, what in (((x.half(),), "fp32 or bf16"), ((x, w[:32]), "shape"), ((x, w.half()), "fp32 or bf16"),
                       ((x, w, w.bfloat16()), "weight is"), ((x, w.cpu()), "tensor on"),
                       ((x[:, :0],), "last dimension"),
                       ((torch.zeros(2, 16385, device=gpu_device),), "width"),
                       ((torch.zeros(2, 4097, device=gpu_device),), "width")):
        with pytest.raises(ValueError, match=what):
            layer_norm(*args)
    stats = torch.zeros(4, 2, device=gpu_device)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(_lib.lib().bioemu_layer_norm_bwd(x.data_ptr(), x.data_ptr(), stats.data_ptr(), None, None,
                                                    w.data_ptr(), None, None, 0, 4, 64, 64, 64, 1, 0, None), "bwd")


def test_gradients_are_first_order(gpu_device):
    x = torch.randn(4, 64, device=gpu_device, requires_grad=True)
    y = layer_norm(x, torch.ones(64, device=gpu_device))
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.sum(), x)


def test_a_leaf_that_wants_its_gradient_accumulated(gpu_device):
    """backward() twice: gradients add up, the op's outputs are not overwritten."""
    x = torch.randn(30, 64, device=gpu_device, requires_grad=True)
    w = torch.ones(64, device=gpu_device, requires_grad=True)
    layer_norm(x, w).square().sum().backward()
    once = x.grad.clone(), w.grad.clone()
    layer_norm(x, w).square().sum().backward()
    assert torch.equal(x.grad, 2 * once[0]) and torch.equal(w.grad, 2 * once[1])


def test_fake_tensors_and_schema(gpu_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(3, 5, 64, device="cuda", dtype=BF16, requires_grad=True)
        w = torch.empty(64, device="cuda", requires_grad=True)
        y = layer_norm(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == x.shape and dx.dtype == BF16 and dw.shape == (64,) and dw.dtype == F32
