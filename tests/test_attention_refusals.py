"""What the entry points between the projections refuse, before anything touches a device (so this runs on a CPU host)."""
import ctypes

import pytest
import torch

from sensenova_u1_amd import PagedKVCache, RotaryTable, ops, paged_attention, prompt_attention, rotary
from sensenova_u1_amd.attention import _CacheStruct, _TableStruct

E_TYPE, E_SHAPE, E_NULL, E_ALIGN = -1, -2, -3, -4
_BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(_BUF) + 63) // 64 * 64
NAN, INF = float("nan"), float("inf")


def _cache(k=P, v=P, ks=P, vs=P, pages=4, page=16, heads=2, dim=64, qt=ops.Q8_0):
    return _CacheStruct(k, v, ks, vs, pages, page, heads, dim, qt)


def _table(turns=P, pairs=16, magnitude=1.0, interleaved=0):
    return _TableStruct(turns, pairs, magnitude, interleaved)


def _at(s):
    return None if s is None else ctypes.addressof(s)


def _rotary(table=_table(), positions=P, tokens=3, dim=64, q=P, heads=2, out=P, k=P, k_heads=1, k_out=P):
    return ops.load_library().sngguf_rotary(_at(table), positions, tokens, dim, q, heads, 64, 64, out, 64, 64, k, k_heads, 64, 64, k_out, 64, 64, None)


def test_rotary_refusals():
    assert _rotary(table=None) == E_NULL
    assert _rotary(positions=None) == E_NULL
    assert _rotary(table=_table(turns=None)) == E_NULL
    for bad in (dict(pairs=0), dict(pairs=33), dict(magnitude=NAN), dict(magnitude=INF)):
        assert _rotary(table=_table(**bad)) == E_SHAPE
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(dim=60), dict(dim=1032), dict(heads=0), dict(heads=65536), dict(k_heads=-1)):
        assert _rotary(**bad) == E_SHAPE
    for bad in (dict(q=None), dict(out=None), dict(k=None), dict(k_out=None)):
        assert _rotary(**bad) == E_NULL
    for bad in (dict(q=P + 1), dict(k_out=P + 1), dict(positions=P + 4), dict(table=_table(turns=P + 4))):
        assert _rotary(**bad) == E_ALIGN
    assert _rotary(tokens=0, q=None, out=None, k=None, k_out=None, positions=None) == 0


BAD_CACHES = [(dict(qt=2), E_TYPE), (dict(pages=0), E_SHAPE), (dict(pages=1 << 31), E_SHAPE), (dict(page=8), E_SHAPE), (dict(page=48), E_SHAPE), (dict(page=8192), E_SHAPE),
              (dict(heads=0), E_SHAPE), (dict(dim=16), E_SHAPE), (dict(dim=80), E_SHAPE), (dict(dim=288), E_SHAPE), (dict(k=None), E_NULL), (dict(v=None), E_NULL),
              (dict(ks=None), E_NULL), (dict(vs=None), E_NULL), (dict(k=P + 8), E_ALIGN), (dict(vs=P + 2), E_ALIGN)]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_refusals(bad, code):
    lib = ops.load_library()
    c = _cache(**bad)
    assert lib.sngguf_cache_write(_at(c), P, 128, 64, P, 128, 64, P, 1, None) == code
    assert lib.sngguf_cache_read(_at(c), P, 1, P, P, None) == code
    t = _table()
    assert lib.sngguf_cache_write_rotary(_at(c), _at(t), P, P, 4, 256, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 1, None) == code
    assert lib.sngguf_paged_attention(P, 1, 4, 256, 64, _at(c), P, 4, 4, P, None, 1, 1, 1.0, 0, P, 256, 64, None, 0, None) == code


def test_cache_call_refusals():
    lib = ops.load_library()
    c, t = _cache(), _table()
    assert lib.sngguf_cache_write(None, P, 128, 64, P, 128, 64, P, 1, None) == E_NULL
    assert lib.sngguf_cache_write(_at(c), P, 128, 64, P, 128, 64, P, -1, None) == E_SHAPE
    for args, code in (((None, P, P), E_NULL), ((P, None, P), E_NULL), ((P, P, None), E_NULL), ((P + 1, P, P), E_ALIGN), ((P, P, P + 4), E_ALIGN)):
        k, v, slots = args
        assert lib.sngguf_cache_write(_at(c), k, 128, 64, v, 128, 64, slots, 1, None) == code
    assert lib.sngguf_cache_write(_at(c), None, 0, 0, None, 0, 0, None, 0, None) == 0
    assert lib.sngguf_cache_read(_at(c), P, 1, None, P, None) == E_NULL
    assert lib.sngguf_cache_read(_at(c), P, 1, P + 2, P, None) == E_ALIGN
    assert lib.sngguf_cache_read(_at(c), P, -1, P, P, None) == E_SHAPE
    assert lib.sngguf_cache_read(_at(c), None, 0, None, None, None) == 0
    wide = _table(pairs=33)
    assert lib.sngguf_cache_write_rotary(_at(c), _at(wide), P, P, 4, 256, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 1, None) == E_SHAPE
    assert lib.sngguf_cache_write_rotary(_at(c), None, P, P, 4, 256, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 1, None) == E_NULL
    assert lib.sngguf_cache_write_rotary(_at(c), _at(t), P, None, 4, 256, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 1, None) == E_NULL
    assert lib.sngguf_cache_write_rotary(_at(c), _at(t), P, P, 0, 256, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, 1, None) == E_SHAPE
    assert lib.sngguf_cache_write_rotary(_at(c), _at(t), None, None, 4, 0, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, None) == 0


def _attention(q=P, tokens=4, heads=4, kv_heads=2, dim=64, k=P, v=P, keys=4, ends_q=P, ends_k=P, n=1, scale=0.1, causal=1, window=0, out=P, ws=None, nbytes=0,
               kt=128, qt=256, qh=64):
    return ops.load_library().sngguf_attention(q, tokens, heads, qt, qh, k, kt, 64, v, 128, 64, keys, kv_heads, dim, ends_q, ends_k, n, scale, causal, window, out, 256, 64,
                                               ws, nbytes, None)


def test_attention_refusals():
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(tokens=1 << 30, heads=4, kv_heads=2), dict(keys=-1), dict(keys=(1 << 31) - 1), dict(n=-1), dict(heads=3), dict(heads=0), dict(kv_heads=0),
                dict(dim=80), dict(dim=16), dict(dim=288), dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(window=-1),
                dict(window=5, causal=0), dict(kt=1 << 26), dict(kt=-128)):
        assert _attention(**bad) == E_SHAPE, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(ends_q=None), dict(ends_k=None)):
        assert _attention(**bad) == E_NULL, bad
    for bad in (dict(q=P + 2), dict(k=P + 8), dict(out=P + 2), dict(ends_q=P + 2), dict(qt=252), dict(qh=66), dict(ws=P + 8, nbytes=64)):
        assert _attention(**bad) == E_ALIGN, bad
    assert _attention(tokens=0, q=None) == 0 and _attention(n=0, ends_q=None) == 0
    lib = ops.load_library()
    assert lib.sngguf_attention_workspace_bytes(0, 9, 1, 4, 2, 64) == 0 and lib.sngguf_attention_workspace_bytes(4, 9, 1, 4, 3, 64) == 0
    assert lib.sngguf_attention_workspace_bytes(1 << 20, 1 << 20, 1, 32, 8, 128) == 0 and lib.sngguf_attention_workspace_bytes(64, 5000, 1, 32, 8, 128) > 0
    assert lib.sngguf_attention_workspace_bytes(64, 64, 1, 32, 8, 128) == 0


def _paged(q=P, tokens=2, heads=4, cache=_cache(), table=P, stride=4, width=4, lens=P, ends=None, n=2, max_new=0, scale=0.1, window=0, out=P, ws=None, nbytes=0):
    return ops.load_library().sngguf_paged_attention(q, tokens, heads, 256, 64, _at(cache), table, stride, width, lens, ends, n, max_new, scale, window, out, 256, 64, ws, nbytes,
                                                     None)


def test_paged_attention_refusals():
    for bad in (dict(tokens=-1), dict(tokens=1 << 30), dict(n=-1), dict(heads=3), dict(max_new=-1), dict(scale=0.0), dict(scale=NAN), dict(window=-1), dict(width=-1),
                dict(width=1 << 27, stride=1 << 27), dict(stride=3), dict(tokens=1)):
        assert _paged(**bad) == E_SHAPE, bad
    for bad in (dict(cache=None), dict(q=None), dict(out=None), dict(lens=None), dict(table=None)):
        assert _paged(**bad) == E_NULL, bad
    for bad in (dict(q=P + 2), dict(out=P + 4), dict(table=P + 2), dict(lens=P + 1), dict(ends=P + 2), dict(ws=P + 4)):
        assert _paged(**bad) == E_ALIGN, bad
    assert _paged(tokens=0, n=0, q=None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    ends = torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: prompt_attention(x, x, x, ends), lambda: rotary(x, None, torch.arange(4), None),
                 lambda: RotaryTable(torch.ones(4, dtype=torch.float64)), lambda: RotaryTable.for_model(64, device="cpu"),
                 lambda: PagedKVCache(torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16)),
                 lambda: PagedKVCache.empty(2, 2, 16, 64, device="cpu"), lambda: paged_attention(x, None, None, None)):
        with pytest.raises(ops.SnGgufError):
            call()


def test_rotary_settings_are_checked():
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=64, scaling="other"), dict(rotary_dim=64, factor=0.0), dict(rotary_dim=64, base=1.0),
                dict(rotary_dim=64, scaling="yarn", factor=4.0)):
        with pytest.raises(ops.SnGgufError):
            RotaryTable.for_model(**bad, device="cpu")
