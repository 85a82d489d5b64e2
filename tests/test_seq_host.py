"""Host side of the trainable operators (CPU only): bucket maps, refusals, state dicts, C ABI checks."""

from __future__ import annotations

import math

import pytest
import torch

from bioemu2_amd import _lib
from bioemu2_amd.layer_norm import LayerNorm, layer_norm
from bioemu2_amd.relative_position import RelativePosition, distance_buckets, relative_position


def test_distance_buckets_own_bucket_each():
    assert distance_buckets(3).tolist() == [0, 1, 2, 3, 4, 5, 6]
    assert distance_buckets(0).tolist() == [0]


@pytest.mark.parametrize("radius,nb", [(128, 32), (128, 64), (64, 64), (1000, 128), (16, 64), (200, 4), (512, 256)])
def test_distance_buckets_log_borders_are_exact(radius, nb):
    """Bucket k of the far distances starts at the least d with (d / exact)^steps >= (radius / exact)^k, in whole
    numbers; both directions alike; offset 0 among the positive ones."""
    m = distance_buckets(radius, nb).tolist()
    half, exact = nb // 2, nb // 4
    steps = half - exact
    assert len(m) == 2 * radius + 1 and m[radius] == 0
    for d in range(1, radius + 1):
        if d < exact:
            want = d
        else:
            k = max(k for k in range(steps + 1) if d ** steps * exact ** k >= radius ** k * exact ** steps)
            want = min(half - 1, exact + k)
        assert m[radius + d] == want and m[radius - d] == half + want, d


def test_distance_buckets_refusals():
    for args in ((-1,), (128,), (128, 6), (128, 260), (5, 64)):
        with pytest.raises(ValueError):
            distance_buckets(*args)


def test_cpu_tensors_are_rejected():
    x = torch.randn(2, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        LayerNorm(8)(x)
    pos = torch.arange(4)[None]
    with pytest.raises(RuntimeError, match="no CPU path"):
        relative_position(x, distance_buckets(0), pos)
    with pytest.raises(RuntimeError, match="no CPU path"):
        RelativePosition(8)(pos)
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm(9)(x)
    with pytest.raises(ValueError, match="at most 256"):
        RelativePosition(8, radius=127, num_buckets=None) and RelativePosition(8, radius=200)


def test_layer_norm_c_abi_refusals():
    lib = _lib.lib()
    assert lib.bioemu_layer_norm_fwd(None, None, None, None, None, 4, 64, 64, 1e-5, 1, 0, None) == -1
    assert b"null" in lib.bioemu_last_error()
    assert lib.bioemu_layer_norm_fwd(None, None, None, None, None, 4, 0, 0, 1e-5, 1, 0, None) == -1
    assert lib.bioemu_layer_norm_fwd(16, None, None, 16, None, 4, 16388, 16388, 1e-5, 1, 0, None) == -2
    assert lib.bioemu_layer_norm_fwd(None, None, None, None, None, 0, 64, 64, 1e-5, 1, 0, None) == 0
    assert lib.bioemu_layer_norm_bwd(16, 16, 16, None, 16, 16, None, None, 0, 4, 64, 64, 64, 1, 0, None) == -3
    assert lib.bioemu_layer_norm_bwd(16, 16, 16, None, 16, None, None, None, 0, 0, 64, 64, 64, 1, 0, None) == -1
    assert lib.bioemu_layer_norm_bwd_workspace_bytes(1 << 20, 128) == 1024 * 2 * 128 * 4
    assert lib.bioemu_layer_norm_bwd_workspace_bytes(0, 128) == 0


def test_relpos_c_abi_refusals():
    lib = _lib.lib()
    assert lib.bioemu_relpos_fwd(None, None, None, None, None, None, 1, 8, 16, 2, 5, 1, 0, None) == -1
    assert lib.bioemu_relpos_fwd(16, 16, 16, None, None, 16, 1, 8, 16, 2, 257, 1, 0, None) == -2
    assert lib.bioemu_relpos_fwd(16, 16, 16, None, None, 16, 1, 8, 16, 2, 0, 1, 0, None) == -1
    assert lib.bioemu_relpos_fwd(16, 16, 16, None, None, 16, 0, 8, 16, 2, 5, 1, 0, None) == 0
    assert lib.bioemu_relpos_bwd(16, 16, 16, None, 16, None, 0, 1, 8, 16, 2, 5, 1, 0, None) == -3
    assert lib.bioemu_relpos_bwd_workspace_bytes(0, 8, 16, 5) == 0
    assert math.prod((1, 5, 16, 4)) == lib.bioemu_relpos_bwd_workspace_bytes(1, 8, 16, 5)


def _attention_args(**over):
    vals = dict(q=16, k=16, v=16, q_batch=128, q_row=32, q_head=16, k_batch=128, k_row=32, k_head=16, v_batch=128,
                v_row=32, v_head=16, q_segments=None, k_segments=None, prefix=None, lengths=None, bias_table=None,
                bias_buckets=None, B=1, Nq=4, Nk=4, H=2, Hk=2, D=16, radius=0, num_buckets=0, scale=0.25, cap=0.0,
                causal=0, f32=1, table_bf16=0) | over
    return _lib.AttentionArgs(**vals)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), -1), (dict(q=8), -1), (dict(k_row=30), -1), (dict(k_row=8), -2), (dict(v_row=1 << 24), -2),
    (dict(D=12), -2), (dict(D=136), -2), (dict(H=3), -1), (dict(H=0), -1), (dict(Nq=1 << 28), -2), (dict(cap=-1.0), -1),
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_segments=16), -1), (dict(bias_table=16), -1),
    (dict(bias_table=16, bias_buckets=16, radius=513, num_buckets=4), -2),
    (dict(bias_table=16, bias_buckets=16, radius=5, num_buckets=257), -2), (dict(B=1 << 20, H=4, Hk=2), -2)])
def test_attention_c_abi_refusals(over, code):
    lib = _lib.lib()
    args = _attention_args(**over)
    assert lib.bioemu_attention_fwd(args, 16, None, None, None, 0, None) == code
    assert lib.bioemu_attention_workspace_bytes(args) == 0
    assert lib.bioemu_attention_bwd_workspace_bytes(args, 0) == 0


def test_attention_c_abi_workspace_and_outputs():
    lib = _lib.lib()
    assert lib.bioemu_attention_fwd(None, 16, None, None, None, 0, None) == -1
    assert lib.bioemu_attention_fwd(_attention_args(), None, None, None, None, 0, None) == -1
    assert lib.bioemu_attention_fwd(_attention_args(B=0), None, None, None, None, 0, None) == 0
    assert lib.bioemu_attention_fwd(_attention_args(), 16, 16, None, None, 0, None) == -1   # o_lo of an fp32 call
    strides = (_lib._c_int64 * 3)(128, 32, 16)
    args = _attention_args()
    assert lib.bioemu_attention_bwd(args, 16, None, 16, 16, strides, 16, 16, 16, None, None, 0, None) == -3
    assert lib.bioemu_attention_bwd(args, 16, None, 16, 16, strides, 16, 16, None, None, 16, 1 << 20, None) == -1
    assert lib.bioemu_attention_bwd(args, 16, None, 16, 16, strides, 16, 16, 16, 16, 16, 1 << 20, None) == -1   # no table
    assert lib.bioemu_attention_bwd_workspace_bytes(args, 0) == 256   # 2 x 1 x 2 x 4 row values, rounded up


def test_attention_rejects_cpu_tensors():
    from bioemu2_amd.attention import SequenceAttention, attention

    q = torch.randn(1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        attention(q, q, q)
    mod = SequenceAttention(2, radius=4)
    assert set(mod.state_dict()) == {"bias"} and mod.bias.shape == (9, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mod(q, q, q)


def _op_calls():
    """name -> (call on meta tensors, its differentiable inputs)."""
    op = {n: _lib.torch_op(n) for n in ("layer_norm", "relative_position", "attention")}
    meta = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="meta")  # noqa: E731
    buckets, positions = meta(5, dtype=torch.uint8), meta(1, 4, dtype=torch.int32)
    return {
        "layer_norm": (lambda x, w, b: op["layer_norm"](x, w, b, 1e-5), [meta(4, 8), meta(8), meta(8)]),
        "relative_position": (lambda t, z: op["relative_position"](t, z, buckets, positions, None, torch.float32),
                              [meta(6, 8), meta(1, 4, 4, 8)]),
        "attention": (lambda q, k, v, t: op["attention"](q, k, v, t, buckets, None, None, None, None, 1.0, 0.0, False),
                      [meta(1, 4, 2, 8) for _ in range(3)] + [meta(5, 2)]),
    }


@pytest.mark.parametrize("name", ["layer_norm", "relative_position", "attention"])
@pytest.mark.parametrize("train", [False, True])
def test_forward_mode_derivatives_are_refused(name, train):
    """A tangent on any input raises, with and without gradients; it is never dropped."""
    import torch.autograd.forward_ad as fw

    call, inputs = _op_calls()[name]
    assert call(*inputs).shape is not None
    for n, t in enumerate(inputs):
        with fw.dual_level():
            args = list(inputs)
            args[n] = fw.make_dual(t.clone().requires_grad_(train), torch.zeros_like(t))
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call(*args)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call(*args)
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(call, tuple(inputs), tuple(inputs))


@pytest.mark.parametrize("name", ["layer_norm", "relative_position", "attention"])
def test_functional_gradients_are_refused(name):
    """torch.func.grad and vjp do not see the gradients; they raise."""
    call, inputs = _op_calls()[name]
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: call(x, *inputs[1:]).sum())(inputs[0])


def test_layer_norm_without_channels_is_refused():
    """Zero channels (or none) raise, in traced calls and in their gradients too, where rows are counted by division."""
    norm, back = _lib.torch_op("layer_norm"), _lib.torch_op("layer_norm_backward")
    for shape in ((2, 0), (0,), ()):
        for train in (False, True):
            x = torch.empty(shape, device="meta", requires_grad=train)
            with pytest.raises(ValueError, match="last dimension"):
                norm(x, None, None, 1e-5)
    x = torch.empty(0, 8, device="meta", requires_grad=True)
    assert torch.autograd.grad(norm(x, None, None, 1e-5).sum(), x)[0].shape == (0, 8)
    x = torch.empty(2, 0, device="meta")
    with pytest.raises(ValueError, match="last dimension"):
        back(x, x, torch.empty(2, 2, device="meta"), None, True, False, False, False)
