"""Calls of more threads than a launch numbers are refused before they are launched (on the CPU: nothing is)."""
import ctypes

import pytest

from sensenova_u1_amd import ops
from sensenova_u1_amd.attention import _CacheStruct, _TableStruct

E_SHAPE = -2
_BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(_BUF) + 63) // 64 * 64


def _at(s):
    return ctypes.addressof(s)


@pytest.mark.parametrize("heads,dim,tokens", [(8, 128, 1 << 25), (1, 32, 1 << 30), (65535, 256, 1 << 20), (8, 256, (1 << 31) - 1)])
def test_cache_read(heads, dim, tokens):
    c = _CacheStruct(P, P, P, P, 1 << 20, 64, heads, dim, ops.Q8_0)
    assert ops.load_library().sngguf_cache_read(_at(c), P, tokens, P, P, None) == E_SHAPE


@pytest.mark.parametrize("heads,tokens", [(40, 1 << 24), (40, (1 << 31) - 1), (1, (1 << 28) + 8)])
def test_rotary_and_writes(heads, tokens):
    lib, t = ops.load_library(), _TableStruct(P, 16, 1.0, 0)
    assert lib.sngguf_rotary(_at(t), P, tokens, 64, P, heads, 64 * heads, 64, P, 64 * heads, 64, None, 0, 0, 0, None, 0, 0, None) == E_SHAPE
    c = _CacheStruct(P, P, P, P, 1 << 20, 64, 16, 128, ops.Q8_0)
    assert lib.sngguf_cache_write(_at(c), P, 2048, 128, P, 2048, 128, P, tokens, None) == E_SHAPE
    assert lib.sngguf_cache_write_rotary(_at(c), _at(t), P, P, heads, 128 * heads, 128, P, 128 * heads, 128, P, 2048, 128, P, 2048, 128, P, tokens, None) == E_SHAPE


def test_attention():
    lib = ops.load_library()
    # 65535 heads of their own keys: a workgroup each for 128 or 256 rows
    assert lib.sngguf_attention(P, 1 << 20, 65535, 65536 * 64, 64, P, 4096, 64, P, 4096, 64, 1 << 20, 65535, 64, P, P, 1, 0.1, 1, 0, P, 65536 * 64, 64, None, 0, None) == E_SHAPE
    c = _CacheStruct(P, P, P, P, 1 << 20, 64, 512, 64, ops.Q8_0)
    for tokens, max_new in ((1 << 15, 1), (1 << 22, 1 << 20)):
        assert lib.sngguf_paged_attention(P, tokens, 512, 512 * 64, 64, _at(c), P, 4, 4, P, P, 1 << 15, max_new, 0.1, 0, P, 512 * 64, 64, None, 0, None) == E_SHAPE
