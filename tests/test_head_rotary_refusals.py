"""What the entry points of normed heads and several positions refuse, before anything touches a device (so this runs on a CPU host)."""
import ctypes

import pytest
import torch

from sensenova_u1_amd import HeadNorm, RotaryAxes, ops
from sensenova_u1_amd.attention import _AXES, _NORM, _CacheStruct

from .test_kept_memory import Standing

E_TYPE, E_SHAPE, E_NULL, E_ALIGN = -1, -2, -3, -4
_BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(_BUF) + 63) // 64 * 64
NAN, INF = float("nan"), float("inf")


def _axes(turns=P, axis=P, pairs=16, magnitude=1.0, interleaved=0, parts=2, part=(16, 16, 0, 0)):
    return _AXES.pack(turns or 0, axis or 0, pairs, magnitude, interleaved, parts, *part)


def _norm(weight=(P, P, None, None), elements=(32, 32, 0, 0), parts=2, kind=2, eps=1e-6):
    return _NORM.pack(*(w or 0 for w in weight), *elements, parts, kind, eps)


def _at(s):
    return s if s is None or isinstance(s, bytes) else ctypes.addressof(s)


def _rotary(table=_axes(), positions=P, axes=3, tokens=3, dim=64, q_norm=_norm(), k_norm=_norm(), q=P, heads=2, out=P, k=P, k_heads=1, k_out=P):
    return ops.load_library().sngguf_head_rotary(_at(table), positions, axes, 3, tokens, dim, _at(q_norm), q, heads, 64, 64, out, 64, 64, _at(k_norm), k, k_heads, 64, 64,
                                                 k_out, 64, 64, None)


def _write(cache=_CacheStruct(P, P, P, P, 4, 16, 1, 64, ops.Q8_0), table=_axes(), positions=P, axes=3, q_norm=_norm(), k_norm=_norm(), q=P, heads=2, out=P, k=P, v=P, slots=P, tokens=3):
    return ops.load_library().sngguf_cache_write_head_rotary(_at(cache), _at(table), positions, axes, 3, _at(q_norm), q, heads, 64, 64, out, 64, 64, _at(k_norm), k, 64, 64,
                                                             v, 64, 64, slots, tokens, None)


BAD_TABLES = [(dict(pairs=0), E_SHAPE), (dict(pairs=33), E_SHAPE), (dict(magnitude=NAN), E_SHAPE), (dict(magnitude=INF), E_SHAPE), (dict(parts=0), E_SHAPE), (dict(parts=5), E_SHAPE),
              (dict(part=(16, 14, 0, 0)), E_SHAPE), (dict(part=(15, 17, 0, 0)), E_SHAPE), (dict(part=(32, 0, 0, 0)), E_SHAPE), (dict(part=(34, -2, 0, 0)), E_SHAPE),
              (dict(turns=None), E_NULL), (dict(turns=P + 4), E_ALIGN), (dict(axis=P + 2), E_ALIGN)]
BAD_NORMS = [(dict(kind=1), E_TYPE), (dict(parts=0), E_SHAPE), (dict(parts=5), E_SHAPE), (dict(eps=-1.0), E_SHAPE), (dict(eps=NAN), E_SHAPE), (dict(eps=INF), E_SHAPE),
             (dict(elements=(32, 24, 0, 0)), E_SHAPE), (dict(elements=(36, 28, 0, 0)), E_SHAPE), (dict(elements=(64, 0, 0, 0)), E_SHAPE), (dict(elements=(72, -8, 0, 0)), E_SHAPE),
             (dict(weight=(P, None, None, None)), E_NULL), (dict(weight=(P, P + 8, None, None)), E_ALIGN)]


@pytest.mark.parametrize("bad,code", BAD_TABLES)
def test_tables(bad, code):
    assert _rotary(table=_axes(**bad)) == code and _write(table=_axes(**bad)) == code


@pytest.mark.parametrize("bad,code", BAD_NORMS)
def test_norms(bad, code):
    assert _rotary(q_norm=_norm(**bad)) == code and _rotary(k_norm=_norm(**bad)) == code
    assert _write(q_norm=_norm(**bad)) == code and _write(k_norm=_norm(**bad)) == code


def test_calls():
    assert _rotary(table=None) == E_NULL and _write(table=None) == E_NULL and _write(cache=None) == E_NULL
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(dim=60), dict(dim=520), dict(heads=0), dict(heads=65536), dict(k_heads=-1), dict(axes=0), dict(axes=1 << 31)):
        assert _rotary(**bad) == E_SHAPE, bad
    for bad in (dict(positions=None), dict(q=None), dict(out=None), dict(k=None), dict(k_out=None)):
        assert _rotary(**bad) == E_NULL, bad
    for bad in (dict(q=P + 1), dict(k_out=P + 1), dict(positions=P + 4)):
        assert _rotary(**bad) == E_ALIGN, bad
    for bad, code in ((dict(tokens=-1), E_SHAPE), (dict(axes=0), E_SHAPE), (dict(heads=0), E_SHAPE), (dict(slots=None), E_NULL), (dict(v=None), E_NULL), (dict(slots=P + 4), E_ALIGN)):
        assert _write(**bad) == code, bad
    assert _rotary(tokens=0, q=None, out=None, k=None, k_out=None, positions=None) == 0 and _write(tokens=0, q=None, out=None, k=None, v=None, slots=None, positions=None) == 0
    # more tokens than a launch has threads for
    assert _rotary(tokens=(1 << 31) - 1, dim=512, table=_axes(pairs=256, parts=1, part=(512, 0, 0, 0)), q_norm=None, k_norm=None, heads=8) == E_SHAPE


def test_host_tensors():
    for call in (lambda: HeadNorm(torch.ones(64)), lambda: HeadNorm(), lambda: RotaryAxes(torch.ones(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32)),
                 lambda: RotaryAxes.for_model([(64, 0, 1e4)], device="cpu")):
        with pytest.raises(ops.SnGgufError):
            call()


@pytest.mark.parametrize("parts", [[], [(63, 0, 1e4)], [(0, 0, 1e4)], [(64, 0, 1.0)]])
def test_settings(parts):
    with pytest.raises(ops.SnGgufError, match="are not known"):
        RotaryAxes.for_model(parts, device="cpu")


def test_the_packed_structures_are_those_of_the_header():
    class Axes(ctypes.Structure):
        _fields_ = [("turns", ctypes.c_void_p), ("axis", ctypes.c_void_p), ("pairs", ctypes.c_int64), ("magnitude", ctypes.c_double), ("interleaved", ctypes.c_int32),
                    ("parts", ctypes.c_int32), ("part", ctypes.c_int32 * 4)]

    class Norm(ctypes.Structure):
        _fields_ = [("weight", ctypes.c_void_p * 4), ("elements", ctypes.c_int32 * 4), ("parts", ctypes.c_int32), ("weight_type", ctypes.c_int32), ("eps", ctypes.c_float)]

    assert bytes(Axes(5, 7, 3, 1.25, 1, 2, (4, 2, 0, 0))) == _AXES.pack(5, 7, 3, 1.25, 1, 2, 4, 2, 0, 0) and ctypes.sizeof(Axes) == _AXES.size
    assert bytes(Norm((1, 2, 3, 4), (8, 16, 24, 32), 4, 2, 0.5)) == _NORM.pack(1, 2, 3, 4, 8, 16, 24, 32, 4, 2, 0.5) and ctypes.sizeof(Norm) == _NORM.size


@pytest.mark.parametrize("eps", [1e300, 3.5e38, -3.5e38, INF, NAN, -1e-9])
def test_an_eps_that_32_bits_do_not_hold(eps):
    weight = torch.Tensor._make_subclass(Standing, torch.ones(64))
    with pytest.raises(ops.SnGgufError, match="HeadNorm: eps is"):
        HeadNorm(weight, eps=eps)
    assert HeadNorm(weight, eps=3.4028234663852886e38).eps == 3.4028234663852886e38
