"""Host side of rotary positions and the paged cache (CPU only): frequencies, refusals, C ABI checks."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from bioemu2_amd import _lib
from bioemu2_amd.paged_cache import PagedCache, paged_append, paged_attention
from bioemu2_amd.rotary import RotaryPosition, rotary, rotary_frequencies

F64 = torch.float64


def test_frequencies():
    f = rotary_frequencies(8)
    assert f.dtype == F64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=F64), rtol=1e-15, atol=0)
    assert torch.allclose(rotary_frequencies(8, scaling="linear", factor=4.0), f / 4, rtol=1e-15, atol=0)
    long = rotary_frequencies(8, scaling="base", factor=4.0)
    assert long[0] == 1.0 and math.isclose(long[-1], f[-1] / 4, rel_tol=1e-14)
    assert rotary_frequencies(2).tolist() == [1.0] and rotary_frequencies(2, scaling="base", factor=3.0).tolist() == [1.0]


def test_frequencies_by_parts():
    """Pairs that turn more than 32 times over the length keep their frequency, those that turn less than once are
    slowed by the factor, in between linearly in the number of turns."""
    length, factor = 2000, 8.0
    f, g = rotary_frequencies(64), rotary_frequencies(64, scaling="parts", factor=factor, length=length)
    turns = length * f / (2 * math.pi)
    for a, b, t in zip(f.tolist(), g.tolist(), turns.tolist()):
        if t >= 32:
            assert b == a
        elif t <= 1:
            assert math.isclose(b, a / factor, rel_tol=1e-15)
        else:
            keep = (t - 1) / 31
            assert math.isclose(b, a * (keep + (1 - keep) / factor), rel_tol=1e-14)
    assert (turns >= 32).any() and (turns <= 1).any() and ((turns > 1) & (turns < 32)).any()


def test_frequencies_refusals():
    for kw in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=2.0), dict(dim=8, scaling="other"),
               dict(dim=8, scaling="parts", factor=2.0), dict(dim=8, scaling="linear", factor=-1.0),
               dict(dim=8, scaling="parts", factor=2.0, length=100, turns=(3.0, 3.0))):
        with pytest.raises(ValueError):
            rotary_frequencies(**kw)


def test_module_keeps_64_bits():
    m = RotaryPosition(16).to(torch.bfloat16).half()
    assert m.frequencies.dtype == F64 and torch.equal(m.frequencies, rotary_frequencies(16))
    assert not m.state_dict() and not list(m.parameters()) and m.magnitude == 1.0
    assert RotaryPosition(16, scaling="parts", factor=4.0, length=64).magnitude == 0.1 * math.log(4.0) + 1.0
    assert RotaryPosition(16, scaling="parts", factor=4.0, length=64, magnitude=1.0).magnitude == 1.0


def test_cpu_tensors_are_rejected():
    x, f = torch.randn(1, 2, 2, 16), rotary_frequencies(16)
    ints = torch.zeros(1, 1, dtype=torch.int32)
    cache = PagedCache(2, 4, 2, 16, dtype=torch.float32)
    assert cache.keys.shape == (2, 4, 2, 16) and cache.keys.stride() == (128, 16, 64, 1)
    for call in (lambda: rotary(x, None, None, f), lambda: RotaryPosition(16)(x), lambda: cache.append(x, x, ints, ints[0]),
                 lambda: cache.attend(x, ints, ints[0]), lambda: paged_append(cache.keys, cache.values, x, x, ints, ints[0]),
                 lambda: paged_attention(x, cache.keys, cache.values, ints, ints[0])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="neither"):
        rotary(None, None, None, f)


def _rotary(**over):
    vals = dict(q=16, k=16, q_batch=128, q_row=32, q_head=16, k_batch=128, k_row=32, k_head=16, positions=None,
                frequencies=16, B=1, N=4, H=2, Hk=2, D=16, pairs=8, magnitude=1.0, interleaved=0, inverse=0, f32=1) | over
    return _lib.RotaryArgs(**vals)


@pytest.mark.parametrize("over,code", [
    (dict(q=8), -1), (dict(k_row=30), -1), (dict(q_head=2), -1), (dict(D=12), -2), (dict(D=520), -2), (dict(D=0), -1),
    (dict(pairs=9), -1), (dict(pairs=-1), -1), (dict(frequencies=None), -1), (dict(B=-1), -1), (dict(N=1 << 31), -2),
    (dict(B=1 << 16, N=1 << 16), -2), (dict(H=0), -1), (dict(H=1 << 20), -2)])
def test_rotary_c_abi_refusals(over, code):
    lib = _lib.lib()
    assert lib.bioemu_rotary(_rotary(**over), 16, 16, None) == code
    stride = (ctypes.c_int64 * 3)(128, 32, 16)
    assert lib.bioemu_paged_append(_cache(), _rotary(**over), 16, stride, 16, None) == code


def test_rotary_c_abi_outputs():
    lib = _lib.lib()
    assert lib.bioemu_rotary(None, 16, 16, None) == -1
    assert lib.bioemu_rotary(_rotary(), None, 16, None) == -1
    assert lib.bioemu_rotary(_rotary(), 16, 24, None) == -1
    assert lib.bioemu_rotary(_rotary(B=0), None, None, None) == 0
    assert lib.bioemu_rotary(_rotary(q=None, k=None), None, None, None) == 0


def _cache(**over):
    vals = dict(keys=16, values=16, keys_page=256, keys_slot=16, keys_head=64, values_page=256, values_slot=16,
                values_head=64, page_table=16, table_stride=4, lengths=16, counts=None, pages=3, page_size=4,
                table_width=4) | over
    return _lib.PagedCacheArgs(**vals)


def _attention(**over):
    vals = dict(q=16, q_batch=128, q_row=32, q_head=16, B=2, Nq=1, Nk=0, H=2, Hk=2, D=16, radius=0, num_buckets=0,
                scale=0.25, cap=0.0, causal=1, f32=1, table_bf16=0) | over
    return _lib.AttentionArgs(**vals)


CACHE_REFUSALS = [
    (dict(keys=None), -1), (dict(values=8), -1), (dict(keys_page=255), -1), (dict(values_slot=2), -1), (dict(lengths=None), -1),
    (dict(page_table=None), -1), (dict(pages=-1), -1), (dict(page_size=0), -1), (dict(table_width=-1), -1),
    (dict(page_size=1 << 21), -2), (dict(table_width=1 << 26, page_size=4), -2), (dict(pages=1 << 31), -2)]


@pytest.mark.parametrize("over,code", CACHE_REFUSALS)
def test_cache_refusals(over, code):
    lib = _lib.lib()
    stride = (ctypes.c_int64 * 3)(128, 32, 16)
    assert lib.bioemu_paged_append(_cache(**over), _rotary(), 16, stride, 16, None) == code
    assert lib.bioemu_paged_attention(_cache(**over), _attention(), 16, None, 0, None) == code
    assert lib.bioemu_paged_attention_workspace_bytes(_cache(**over), _attention()) == 0


def test_append_refusals():
    lib = _lib.lib()
    stride = (ctypes.c_int64 * 3)(128, 32, 16)
    odd = (ctypes.c_int64 * 3)(126, 32, 16)
    assert lib.bioemu_paged_append(None, _rotary(), 16, stride, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), None, 16, stride, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(k=None), 16, stride, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(), None, stride, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(), 16, None, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(B=2), 16, odd, 16, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(), 16, stride, None, None) == -1
    assert lib.bioemu_paged_append(_cache(), _rotary(N=0), None, None, None, None) == 0


@pytest.mark.parametrize("over,code", [
    (dict(Nk=4), -1), (dict(k=16), -1), (dict(lengths=16), -1), (dict(prefix=16), -1), (dict(D=12), -2), (dict(D=136), -2),
    (dict(H=3), -1), (dict(cap=-1.0), -1), (dict(cap=2e5), -2), (dict(q=8), -1), (dict(q=None), -1),
    (dict(bias_table=16), -1), (dict(Nq=1 << 28), -2)])
def test_attention_refusals(over, code):
    lib = _lib.lib()
    assert lib.bioemu_paged_attention(_cache(), _attention(**over), 16, None, 0, None) == code
    assert lib.bioemu_paged_attention_workspace_bytes(_cache(), _attention(**over)) == 0


def test_attention_workspace_and_outputs():
    lib = _lib.lib()
    assert lib.bioemu_paged_attention(_cache(), _attention(), None, None, 0, None) == -1
    assert lib.bioemu_paged_attention(_cache(), _attention(), 8, None, 0, None) == -1
    assert lib.bioemu_paged_attention(_cache(), _attention(B=0), None, None, 0, None) == 0
    assert lib.bioemu_paged_attention_workspace_bytes(_cache(), _attention()) == 0      # few keys: no parts
    wide = _cache(table_width=1000)
    need = lib.bioemu_paged_attention_workspace_bytes(wide, _attention())
    assert need > 0
    assert lib.bioemu_paged_attention(wide, _attention(), 16, None, 0, None) == -3
    assert lib.bioemu_paged_attention(wide, _attention(), 16, 16, need - 1, None) == -3


def test_forward_derivatives_are_refused():
    import torch.autograd.forward_ad as fw

    op = _lib.torch_op("rotary")
    x, f = torch.empty(1, 2, 2, 16, device="meta"), torch.empty(8, dtype=F64, device="meta")
    assert op(x, None, None, f, False, 1.0, False)[0].shape == x.shape
    with fw.dual_level():
        dual = fw.make_dual(x, torch.zeros_like(x))
        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            op(dual, None, None, f, False, 1.0, False)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint64, torch.uint32, torch.int32, torch.int16, torch.uint8])
def test_numbers_that_32_bits_do_not_hold(dtype):
    """Tables and lengths of 64 bits are taken to the nearest number of 32 bits: 2^32 names no page, not the first."""
    from bioemu2_amd.paged_cache import _ints

    info = torch.iinfo(dtype)
    want = [0, 3, 100, max(info.min, -2 ** 31), min(info.max, 2 ** 31 - 1)]
    have = [0, 3, 100, info.min, info.max if dtype != torch.uint64 else 2 ** 63 - 1]
    if info.bits == 64:
        have += [2 ** 32, 2 ** 32 + 3, 2 ** 31]
        want += [2 ** 31 - 1] * 3
    for t in _ints("here", *[torch.tensor(have, dtype=dtype)] * 3):
        assert t.dtype == torch.int32 and t.tolist() == want
    table = torch.tensor([have, have], dtype=dtype).T
    assert _ints("here", table, table[:, 0], None)[0].tolist() == [[w, w] for w in want]
    with pytest.raises(ValueError, match="whole numbers"):
        _ints("here", table.float(), table[:, 0], None)


@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=3.0), dict(scaling="base", factor=3.0),
                                dict(scaling="parts", factor=8.0, length=2000, turns=(2.0, 20.0))], ids=str)
def test_module_made_without_values(kw):
    """Built on the meta device, the module has its frequencies once it is brought to another."""
    want = RotaryPosition(32, base=5000.0, **kw).frequencies
    assert torch.equal(want, rotary_frequencies(32, 5000.0, **kw)) and want.device.type == "cpu"
    with torch.device("meta"):
        m = RotaryPosition(32, base=5000.0, **kw)
    assert m.frequencies.is_meta and m.frequencies.shape == (16,)
    got = m.to_empty(device="cpu").frequencies
    assert got.dtype == F64 and torch.equal(got, want)
    m = RotaryPosition(32, base=5000.0, **kw).to("meta")
    assert m.frequencies.is_meta and torch.equal(m.to_empty(device="cpu").half().frequencies, want)
    both = torch.nn.ModuleList([torch.nn.Linear(2, 2, device="meta"), m.to("meta")]).to_empty(device="cpu")
    assert torch.equal(both[1].frequencies, want)


def test_as_many_rows_as_a_launch_has_threads_for():
    """2^24 - 4 blocks of 32 rows, a workgroup of 256 threads each and rounded up to 8, would be 2^32 threads."""
    lib = _lib.lib()
    many = dict(B=69, Nq=89 * 683 * 128, H=1, Hk=1, D=8, q_batch=8 * 89 * 683 * 128, q_row=8, q_head=8)
    assert 69 * many["Nq"] // 32 == (1 << 24) - 4
    assert lib.bioemu_paged_attention(_cache(), _attention(**many), 16, None, 0, None) == -2
    assert b"too many" in lib.bioemu_last_error()
    assert lib.bioemu_paged_attention_workspace_bytes(_cache(), _attention(**many)) == 0
