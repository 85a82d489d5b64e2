"""Trainable torch ops over the C ABI: LayerNorm, relative positions, attention.

As ``_ops``: ``launch_*`` functions validate tensors and call the C ABI on the
current HIP stream of the tensors' device with caller-provided outputs, and
``torch.ops.bioemu_mi355x.*`` are ``torch.library`` custom ops (HIP only) with a
registered gradient.  A plain call does not pass the dispatcher: without
gradients it reaches the body, with them one ``autograd.Function``.  Gradients
are first order.
"""

from __future__ import annotations

import ctypes
import struct

import torch
from torch import Tensor

from ._lib import AttentionArgs, check, lib
from ._ops import BF16, F32, _check_tensor, _Op, _ptr, _stream, _unobserved, require_gpu, workspace

_TYPES = (BF16, F32)
_current_device = torch._C._cuda_getDevice


def _call(t: Tensor, what: str, *args) -> None:
    """The C ABI's ``what`` on t's device (current or not) and its current stream."""
    fn = getattr(lib(), what)
    if _current_device() == t.get_device():
        rc = fn(*args, _stream(t))
    else:
        with torch.cuda.device(t.device):
            rc = fn(*args, _stream(t))
    if rc:
        check(rc, what)


class _TrainOp(_Op):
    """An ``_Op`` with a gradient.  ``save`` takes (ctx, args, outputs), ``grad`` (ctx, gradients of the outputs).  The
    op's last argument says whether a gradient is wanted (what the backward pass reads is not written by a serving
    call) and is filled in here; callers get the first output."""

    def __init__(self, name: str, body, save, grad):
        super().__init__(name, body)
        self.op.register_autograd(grad, setup_context=lambda ctx, inputs, output: save(ctx, inputs, output))
        once = torch.autograd.function.once_differentiable(lambda ctx, g: grad(ctx, g, None))

        def forward(ctx, *args):
            out = body(*args)
            save(ctx, args, out)
            return out[0]

        def backward(ctx, g):
            # grad mode is off but where a graph of the gradient is asked for, which there is none of
            return once(ctx, g) if torch.is_grad_enabled() else grad(ctx, g, None)

        self.fn = type(name, (torch.autograd.Function,),
                       {"forward": staticmethod(forward), "backward": staticmethod(backward)})

    def __call__(self, *args):
        train = False
        if torch.is_grad_enabled():
            for a in args:
                if isinstance(a, Tensor) and a.requires_grad:
                    train = True
                    break
        if _unobserved(args) and self._own():
            return self.fn.apply(*args, True) if train else self.body(*args, False)[0]
        return self.op(*args, train)[0]


def _param_type(t: Tensor | None, what: str, shape: tuple[int, ...], device) -> int:
    """1 for bf16 and 0 for fp32 parameters."""
    if t is None:
        return 0
    if t.dtype not in _TYPES:
        raise ValueError(f"{what}: expected fp32 or bf16, got {t.dtype}")
    _check_tensor(t, what, t.dtype, shape, device)
    return int(t.dtype == BF16)


def _activation(t: Tensor, what: str) -> int:
    """1 for fp32 and 0 for bf16 activations."""
    require_gpu(t, what)
    if t.dtype not in _TYPES:
        raise ValueError(f"{what}: expected fp32 or bf16, got {t.dtype}")
    return int(t.dtype == F32)


# ----------------------------------------------------------------------------
# LayerNorm
# ----------------------------------------------------------------------------
def _as_rows(x: Tensor) -> tuple[Tensor, int]:
    """``x`` with the stride of its rows (of the last dimension, neighbouring values adjacent): itself where its strides
    allow, a copy else."""
    c = x.shape[-1]
    if x.is_contiguous():
        return x, c
    if x.stride(-1) == 1 or c == 1:
        try:
            rows = x.view(-1, c)
            if rows.stride(1) == 1:
                return rows, rows.stride(0)
        except RuntimeError:
            pass
    return x.contiguous(), c


def _norm_types(x: Tensor, weight: Tensor | None, bias: Tensor | None) -> tuple[int, int]:
    """(1 for fp32 activations, 1 for bf16 parameters)."""
    f32, c = _activation(x, "layer_norm"), x.shape[-1]
    w16 = _param_type(weight, "layer_norm weight", (c,), x.device)
    if bias is None:
        return f32, w16
    if weight is not None and bias.dtype != weight.dtype:
        raise ValueError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    return f32, _param_type(bias, "layer_norm bias", (c,), x.device)


def layer_norm_bwd_workspace_bytes(rows: int, c: int) -> int:
    return int(lib().bioemu_layer_norm_bwd_workspace_bytes(rows, c))


def launch_layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, y: Tensor, eps: float,
                      stats: Tensor | None = None) -> Tensor:
    """LayerNorm of the rows ``x`` [rows, c] (any row stride) into contiguous ``y``; ``stats`` [rows, 2] fp32."""
    if x.ndim != 2 or x.stride(1) != 1:
        raise ValueError("layer_norm: x must be [rows, c] with adjacent values")
    f32, w16 = _norm_types(x, weight, bias)
    rows, c = x.shape
    _check_tensor(y, "layer_norm y", x.dtype, (rows, c), x.device)
    if stats is not None:
        _check_tensor(stats, "layer_norm stats", F32, (rows, 2), x.device)
    _call(x, "bioemu_layer_norm_fwd", x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats), rows, c,
          x.stride(0), eps, f32, w16)
    return y


def launch_layer_norm_bwd(x: Tensor, dy: Tensor, stats: Tensor, weight: Tensor | None, dx: Tensor | None,
                          dweight: Tensor | None, dbias: Tensor | None, ws: Tensor | None = None) -> None:
    """Gradients of ``launch_layer_norm`` into ``dx`` [rows, c], ``dweight``, ``dbias`` (each may be None)."""
    if x.ndim != 2 or x.stride(1) != 1 or dy.shape != x.shape or dy.dtype != x.dtype or dy.stride(1) != 1:
        raise ValueError("layer_norm_bwd: x and dy must be [rows, c] of one type with adjacent values")
    f32, w16 = _norm_types(x, weight, None)
    rows, c = x.shape
    dev = x.device
    _check_tensor(stats, "layer_norm stats", F32, (rows, 2), dev)
    if dx is not None:
        _check_tensor(dx, "layer_norm dx", x.dtype, (rows, c), dev)
    for t in (dweight, dbias):
        if t is not None and weight is not None and t.dtype != weight.dtype:
            raise ValueError("layer_norm_bwd: weight gradients take the weight's type")
        w16 |= _param_type(t, "layer_norm weight gradient", (c,), dev)
    need = layer_norm_bwd_workspace_bytes(rows, c) if dweight is not None or dbias is not None else 0
    if need and (ws is None or ws.numel() < need):
        ws = workspace(need, dev)
    _call(x, "bioemu_layer_norm_bwd", x.data_ptr(), dy.data_ptr(), stats.data_ptr(), _ptr(weight), _ptr(dx),
          _ptr(dweight), _ptr(dbias), _ptr(ws), 0 if ws is None else ws.numel(), rows, c, x.stride(0), dy.stride(0),
          f32, w16)


def _layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, train: bool) -> tuple[Tensor, Tensor]:
    f32, w16 = _norm_types(x, weight, bias)
    src, stride = _as_rows(x)
    c = x.shape[-1]
    rows = x.numel() // c
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((rows if train else 0, 2), dtype=F32, device=x.device)
    _call(x, "bioemu_layer_norm_fwd", src.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(),
          stats.data_ptr() if train else None, rows, c, stride, eps, f32, w16)
    return y, stats


def _layer_norm_backward(x: Tensor, dy: Tensor, stats: Tensor, weight: Tensor | None, want_x: bool, want_w: bool,
                         want_b: bool, bias_bf16: bool) -> tuple[Tensor, Tensor, Tensor]:
    dev, c = x.device, x.shape[-1]
    rows = x.numel() // c
    wt = weight.dtype if weight is not None else (BF16 if bias_bf16 else F32)
    dx = torch.empty(x.shape if want_x else (0,), dtype=x.dtype, device=dev)
    dw = torch.empty((c if want_w else 0,), dtype=wt, device=dev)
    db = torch.empty((c if want_b else 0,), dtype=wt, device=dev)
    if rows == 0:
        return dx, dw.zero_(), db.zero_()
    (src, stride), (dsrc, dstride) = _as_rows(x), _as_rows(dy)
    ws = None
    if want_w or want_b:
        ws = workspace(layer_norm_bwd_workspace_bytes(rows, c), dev)
    _call(x, "bioemu_layer_norm_bwd", src.data_ptr(), dsrc.data_ptr(), stats.data_ptr(), _ptr(weight),
          dx.data_ptr() if want_x else None, dw.data_ptr() if want_w else None, db.data_ptr() if want_b else None,
          _ptr(ws), 0 if ws is None else ws.numel(), rows, c, stride, dstride, int(x.dtype == F32), int(wt == BF16))
    return dx, dw, db


layer_norm_backward = _Op("layer_norm_backward", _layer_norm_backward)


@layer_norm_backward.register_fake
def _(x, dy, stats, weight, want_x, want_w, want_b, bias_bf16):
    wt = weight.dtype if weight is not None else (BF16 if bias_bf16 else F32)
    return (x.new_empty(x.shape if want_x else (0,)), x.new_empty((x.shape[-1] if want_w else 0,), dtype=wt),
            x.new_empty((x.shape[-1] if want_b else 0,), dtype=wt))


def _layer_norm_save(ctx, inputs, output) -> None:
    x, weight, bias, _, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.bias_bf16 = bias is not None and bias.dtype == BF16


def _layer_norm_grad(ctx, dy, _):
    x, weight, stats = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = layer_norm_backward(x, dy, stats, weight, need[0], need[1], need[2], ctx.bias_bf16)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None)


layer_norm = _TrainOp("layer_norm", _layer_norm, _layer_norm_save, _layer_norm_grad)


@layer_norm.register_fake
def _(x, weight, bias, eps, train):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), x.new_empty(
        (x.numel() // x.shape[-1] if train else 0, 2), dtype=F32)


# ----------------------------------------------------------------------------
# Relative positions
# ----------------------------------------------------------------------------
def relpos_bwd_workspace_bytes(B: int, N: int, C: int, num_buckets: int) -> int:
    return int(lib().bioemu_relpos_bwd_workspace_bytes(B, N, C, num_buckets))


def _check_relpos(what: str, buckets: Tensor, positions: Tensor, chains: Tensor | None, dev) -> int:
    if positions.ndim != 2:
        raise ValueError(f"{what}: positions must be [B, N], got {tuple(positions.shape)}")
    _check_tensor(positions, f"{what} positions", torch.int32, tuple(positions.shape), dev)
    if chains is not None:
        _check_tensor(chains, f"{what} chains", torch.int32, tuple(positions.shape), dev)
    if buckets.ndim != 1 or buckets.numel() % 2 == 0:
        raise ValueError(f"{what}: buckets must be [2 * radius + 1], got {tuple(buckets.shape)}")
    _check_tensor(buckets, f"{what} buckets", torch.uint8, tuple(buckets.shape), dev)
    return buckets.numel() // 2


def launch_relpos(table: Tensor, buckets: Tensor, positions: Tensor, chains: Tensor | None, z: Tensor | None,
                  out: Tensor) -> Tensor:
    """``out`` [B, N, N, C] = ``z`` + ``table`` [num_buckets, C] at the buckets of the pairs' offsets."""
    f32 = _activation(out, "relpos")
    radius = _check_relpos("relpos", buckets, positions, chains, out.device)
    (B, N), (NB, C) = positions.shape, table.shape
    t16 = _param_type(table, "relpos table", (NB, C), out.device)
    _check_tensor(out, "relpos out", out.dtype, (B, N, N, C), out.device)
    if z is not None:
        _check_tensor(z, "relpos z", out.dtype, (B, N, N, C), out.device)
    _call(out, "bioemu_relpos_fwd", table.data_ptr(), buckets.data_ptr(), positions.data_ptr(), _ptr(chains), _ptr(z),
          out.data_ptr(), B, N, C, radius, NB, f32, t16)
    return out


def launch_relpos_bwd(dout: Tensor, buckets: Tensor, positions: Tensor, chains: Tensor | None, dtable: Tensor,
                      ws: Tensor | None = None) -> Tensor:
    """``dtable`` [num_buckets, C]: the sums of ``dout`` [B, N, N, C] by bucket."""
    f32 = _activation(dout, "relpos_bwd")
    radius = _check_relpos("relpos_bwd", buckets, positions, chains, dout.device)
    (B, N), (NB, C) = positions.shape, dtable.shape
    _check_tensor(dout, "relpos_bwd dout", dout.dtype, (B, N, N, C), dout.device)
    t16 = _param_type(dtable, "relpos_bwd dtable", (NB, C), dout.device)
    need = relpos_bwd_workspace_bytes(B, N, C, NB)
    if ws is None or ws.numel() < need:
        ws = workspace(need, dout.device)
    _call(dout, "bioemu_relpos_bwd", dout.data_ptr(), buckets.data_ptr(), positions.data_ptr(), _ptr(chains),
          dtable.data_ptr(), ws.data_ptr(), ws.numel(), B, N, C, radius, NB, f32, t16)
    return dtable


def _relative_position(table: Tensor, z: Tensor | None, buckets: Tensor, positions: Tensor, chains: Tensor | None,
                       dtype: torch.dtype, train: bool) -> tuple[Tensor, Tensor]:
    B, N = positions.shape
    out = torch.empty((B, N, N, table.shape[1]), dtype=dtype, device=table.device)
    launch_relpos(table.contiguous(), buckets, positions, chains, None if z is None else z.contiguous(), out)
    return out, table.new_empty((0,))   # a gradient reads no result


def _relative_position_backward(dout: Tensor, buckets: Tensor, positions: Tensor, chains: Tensor | None,
                                num_buckets: int, dtype: torch.dtype) -> Tensor:
    dtable = torch.empty((num_buckets, dout.shape[-1]), dtype=dtype, device=dout.device)
    if dout.numel() == 0:
        return dtable.zero_()
    return launch_relpos_bwd(dout.contiguous(), buckets, positions, chains, dtable)


relative_position_backward = _Op("relative_position_backward", _relative_position_backward)


@relative_position_backward.register_fake
def _(dout, buckets, positions, chains, num_buckets, dtype):
    return dout.new_empty((num_buckets, dout.shape[-1]), dtype=dtype)


def _relative_position_save(ctx, inputs, output) -> None:
    table, _, buckets, positions, chains, _, _ = inputs
    ctx.save_for_backward(buckets, positions, chains)
    ctx.table = table.shape[0], table.dtype


def _relative_position_grad(ctx, dout, _):
    buckets, positions, chains = ctx.saved_tensors
    need = ctx.needs_input_grad
    dtable = relative_position_backward(dout, buckets, positions, chains, *ctx.table) if need[0] else None
    return (dtable, dout if need[1] else None, None, None, None, None, None)


relative_position = _TrainOp("relative_position", _relative_position, _relative_position_save, _relative_position_grad)


@relative_position.register_fake
def _(table, z, buckets, positions, chains, dtype, train):
    B, N = positions.shape
    return table.new_empty((B, N, N, table.shape[1]), dtype=dtype), table.new_empty((0,))


# ----------------------------------------------------------------------------
# Attention
# ----------------------------------------------------------------------------
_MAX_ROW_STRIDE = 1 << 23
_PACKED_ARGS = struct.Struct("@3P9q6P8q2f3i0q").pack   # AttentionArgs, a few times faster than field by field
assert len(_PACKED_ARGS(*[0] * 31)) == ctypes.sizeof(AttentionArgs)


def _heads(t: Tensor) -> Tensor:
    """[B, N, H, D] with adjacent values of a head and rows at 16-byte addresses: ``t`` where it is so, a copy else."""
    b, n, h, d = t.stride()
    _, rows, _, width = t.shape
    per = 16 // t.element_size()
    if (d == 1 and (n >= width or rows <= 1) and n <= _MAX_ROW_STRIDE and not (b % per or n % per or h % per)
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _attention_args(q, k, v, table, buckets, q_segments, k_segments, prefix, lengths, scale: float, cap: float,
                    causal: bool) -> AttentionArgs:
    f32 = _activation(q, "attention")
    dev = q.device
    if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"attention: q is {q.dtype}, k {k.dtype}, v {v.dtype}")
    if k.device != dev or v.device != dev:
        raise ValueError(f"attention: q on {dev}, k on {k.device}, v on {v.device}")
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    if (q_segments is None) != (k_segments is None):
        raise ValueError("attention: segments of queries and of keys come together")
    for t, name, shape in ((q_segments, "segments", (B, Nq)), (k_segments, "key segments", (B, Nk)),
                           (prefix, "prefix", (B,)), (lengths, "cache_lengths", (B,))):
        if t is not None:
            _check_tensor(t, f"attention {name}", torch.int32, shape, dev)
    radius = nb = t16 = 0
    if table is not None:
        if buckets is None or table.ndim != 2:
            raise ValueError("attention: a bias table [num_buckets, H] comes with its buckets")
        if buckets.ndim != 1 or buckets.numel() % 2 == 0:
            raise ValueError(f"attention: buckets must be [2 * radius + 1], got {tuple(buckets.shape)}")
        _check_tensor(buckets, "attention buckets", torch.uint8, tuple(buckets.shape), dev)
        radius, nb = buckets.numel() // 2, table.shape[0]
        t16 = _param_type(table, "attention bias table", (nb, H), dev)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    return AttentionArgs.from_buffer_copy(_PACKED_ARGS(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        _ptr(q_segments) or 0, _ptr(k_segments) or 0, _ptr(prefix) or 0, _ptr(lengths) or 0, _ptr(table) or 0,
        0 if table is None else buckets.data_ptr(), B, Nq, Nk, H, Hk, D, radius, nb, scale, cap, int(causal), f32, t16))


def launch_attention(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor | None = None, *,
                     bias_table: Tensor | None = None, bias_buckets: Tensor | None = None,
                     q_segments: Tensor | None = None, k_segments: Tensor | None = None, prefix: Tensor | None = None,
                     lengths: Tensor | None = None, scale: float, cap: float = 0.0, causal: bool = False,
                     ws: Tensor | None = None) -> Tensor:
    """``out`` [B, Nq, H, D] (contiguous); ``lse`` [B, H, Nq] fp32 is what the backward pass needs."""
    args = _attention_args(q, k, v, bias_table, bias_buckets, q_segments, k_segments, prefix, lengths, scale, cap, causal)
    _check_tensor(out, "attention out", q.dtype, tuple(q.shape), q.device)
    if lse is not None:
        _check_tensor(lse, "attention lse", F32, (q.shape[0], q.shape[2], q.shape[1]), q.device)
    need = lib().bioemu_attention_workspace_bytes(args)
    if need and (ws is None or ws.numel() < need):
        ws = workspace(need, q.device)
    _call(q, "bioemu_attention_fwd", args, out.data_ptr(), _ptr(lse), _ptr(ws), 0 if ws is None else ws.numel())
    return out


def launch_attention_bwd(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, dout: Tensor, dq: Tensor,
                         dk: Tensor, dv: Tensor, dtable: Tensor | None = None, *, bias_table: Tensor | None = None,
                         bias_buckets: Tensor | None = None, q_segments: Tensor | None = None,
                         k_segments: Tensor | None = None, prefix: Tensor | None = None,
                         lengths: Tensor | None = None, scale: float, cap: float = 0.0, causal: bool = False,
                         ws: Tensor | None = None) -> None:
    """Gradients of ``launch_attention`` (contiguous ``dq``, ``dk``, ``dv``; ``dtable`` may be None)."""
    args = _attention_args(q, k, v, bias_table, bias_buckets, q_segments, k_segments, prefix, lengths, scale, cap, causal)
    dev = q.device
    _check_tensor(out, "attention out", q.dtype, tuple(q.shape), dev)
    _check_tensor(lse, "attention lse", F32, (q.shape[0], q.shape[2], q.shape[1]), dev)
    if dout.shape != q.shape or dout.dtype != q.dtype or dout.device != dev or dout.stride(3) != 1:
        raise ValueError(f"attention_bwd: dout {dout.dtype} {tuple(dout.shape)} of q {q.dtype} {tuple(q.shape)}")
    for t, like, name in ((dq, q, "dq"), (dk, k, "dk"), (dv, v, "dv")):
        _check_tensor(t, f"attention {name}", q.dtype, tuple(like.shape), dev)
    if dtable is not None:
        if bias_table is None:
            raise ValueError("attention_bwd: dtable without a bias table")
        _check_tensor(dtable, "attention dtable", bias_table.dtype, tuple(bias_table.shape), dev)
    st = dout.stride()
    need = lib().bioemu_attention_bwd_workspace_bytes(args, int(dtable is not None))
    if ws is None or ws.numel() < need:
        ws = workspace(need, dev)
    _call(q, "bioemu_attention_bwd", args, out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
          (ctypes.c_int64 * 3)(st[0], st[1], st[2]), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dtable),
          ws.data_ptr(), ws.numel())


def _attention(q: Tensor, k: Tensor, v: Tensor, table: Tensor | None, buckets: Tensor | None,
               q_segments: Tensor | None, k_segments: Tensor | None, prefix: Tensor | None, lengths: Tensor | None,
               scale: float, cap: float, causal: bool, train: bool) -> tuple[Tensor, Tensor]:
    require_gpu(q, "attention")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]) if train else (0,), dtype=F32, device=q.device)
    launch_attention(_heads(q), _heads(k), _heads(v), out, lse if train else None, bias_table=table,
                     bias_buckets=buckets, q_segments=q_segments, k_segments=k_segments, prefix=prefix,
                     lengths=lengths, scale=scale, cap=cap, causal=causal)
    return out, lse


def _attention_backward(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, dout: Tensor, table: Tensor | None,
                        buckets: Tensor | None, q_segments: Tensor | None, k_segments: Tensor | None,
                        prefix: Tensor | None, lengths: Tensor | None, scale: float, cap: float, causal: bool,
                        want_table: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    dtable = torch.empty(table.shape if want_table else (0,), dtype=q.dtype if table is None else table.dtype,
                         device=q.device)
    if q.shape[0] == 0 or q.shape[1] == 0:
        return dq, dk.zero_(), dv.zero_(), dtable.zero_()
    launch_attention_bwd(_heads(q), _heads(k), _heads(v), out, lse, _heads(dout), dq, dk, dv,
                         dtable if want_table else None, bias_table=table, bias_buckets=buckets,
                         q_segments=q_segments, k_segments=k_segments, prefix=prefix, lengths=lengths, scale=scale,
                         cap=cap, causal=causal)
    return dq, dk, dv, dtable


attention_backward = _Op("attention_backward", _attention_backward)


@attention_backward.register_fake
def _(q, k, v, out, lse, dout, table, buckets, q_segments, k_segments, prefix, lengths, scale, cap, causal, want_table):
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape),
            table.new_empty(table.shape) if want_table else q.new_empty((0,)))


def _attention_save(ctx, inputs, output) -> None:
    q, k, v, table, buckets, q_segments, k_segments, prefix, lengths, scale, cap, causal, _ = inputs
    ctx.save_for_backward(q, k, v, output[0], output[1], table, buckets, q_segments, k_segments, prefix, lengths)
    ctx.plain = scale, cap, causal


def _attention_grad(ctx, dout, _):
    q, k, v, out, lse, *rest = ctx.saved_tensors
    need = ctx.needs_input_grad
    dq, dk, dv, dtable = attention_backward(q, k, v, out, lse, dout, *rest, *ctx.plain, need[3])
    return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
            dtable if need[3] else None) + (None,) * 9


attention = _TrainOp("attention", _attention, _attention_save, _attention_grad)


@attention.register_fake
def _(q, k, v, table, buckets, q_segments, k_segments, prefix, lengths, scale, cap, causal, train):
    return q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[2], q.shape[1]) if train else (0,), dtype=F32)
