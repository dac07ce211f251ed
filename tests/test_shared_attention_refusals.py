"""What the entry point of sequences that begin alike refuses, before anything touches a device (so this runs on a CPU host)."""
import ctypes

from sensenova_u1_amd import ops
from sensenova_u1_amd.attention import _CacheStruct

E_TYPE, E_SHAPE, E_NULL, E_ALIGN = -1, -2, -3, -4
_BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(_BUF) + 63) // 64 * 64
NAN = float("nan")


def _cache(k=P, pages=4, page=16, heads=2, dim=64, qt=ops.Q8_0):
    return _CacheStruct(k, P, P, P, pages, page, heads, dim, qt)


WIDE = 1 << 16       # pages of a row of the table: enough keys for the groups to count


def _call(q=P, tokens=2, heads=4, cache=_cache(), table=P, stride=WIDE, width=WIDE, lens=P, ends=None, n=2, groups=P, shared=P, count=1, max_new=0, scale=0.1, out=P, ws=P, nbytes=1 << 40, qt=256):
    return ops.load_library().sngguf_shared_attention(q, tokens, heads, qt, 64, None if cache is None else ctypes.addressof(cache), table, stride, width, lens, ends, n, groups, shared,
                                                      count, max_new, scale, out, 256, 64, ws, nbytes, None)


def test_refusals():
    for bad in (dict(tokens=-1), dict(tokens=1 << 30), dict(n=-1), dict(heads=3), dict(max_new=-1), dict(scale=0.0), dict(scale=NAN), dict(width=-1), dict(width=1 << 27, stride=1 << 27),
                dict(stride=WIDE - 1), dict(tokens=1), dict(count=0), dict(count=-1), dict(count=1 << 30), dict(nbytes=0), dict(nbytes=64), dict(cache=_cache(pages=0)), dict(cache=_cache(dim=80))):
        assert _call(**bad) == E_SHAPE, bad
    for bad in (dict(cache=None), dict(q=None), dict(out=None), dict(lens=None), dict(table=None), dict(groups=None), dict(shared=None), dict(ws=None), dict(cache=_cache(k=None))):
        assert _call(**bad) == E_NULL, bad
    for bad in (dict(q=P + 2), dict(out=P + 4), dict(table=P + 2), dict(lens=P + 1), dict(ends=P + 2), dict(groups=P + 2), dict(shared=P + 1), dict(ws=P + 4), dict(qt=252)):
        assert _call(**bad) == E_ALIGN, bad
    assert _call(cache=_cache(qt=2)) == E_TYPE
    assert _call(tokens=0, n=0, q=None, ws=None, nbytes=0) == 0


def test_few_keys_need_no_workspace():
    for bad, code in ((dict(groups=None), E_NULL), (dict(shared=P + 2), E_ALIGN), (dict(count=0), E_SHAPE)):
        assert _call(width=4, stride=4, ws=None, nbytes=0, **bad) == code, bad


def test_workspace():
    lib = ops.load_library()
    size, paged = lib.sngguf_shared_attention_workspace_bytes, lib.sngguf_paged_attention_workspace_bytes
    assert size(64, 64, 1, 1, 16384, 32, 8, 128, ops.BF16) > paged(64, 64, 1, 16384, 32, 8, 128)
    assert size(4, 4, 1, 1, 512, 32, 8, 128, ops.BF16) == paged(4, 4, 1, 512, 32, 8, 128)                     # few keys
    assert size(1024, 4, 1, 256, 65536, 32, 8, 128, ops.BF16) == paged(1024, 4, 256, 65536, 32, 8, 128)       # many rows of each
    for bad in ((0, 1, 1, 1, 64, 4, 2, 64), (4, 0, 1, 1, 64, 4, 2, 64), (4, 1, 0, 1, 64, 4, 2, 64), (4, 1, 1, -1, 64, 4, 2, 64), (4, 1, 1, 1, -1, 4, 2, 64), (4, 1, 1, 1, 64, 4, 3, 64),
                (4, 1, 1, 1, 64, 4, 2, 80), (4, 1, 1, 1, 1 << 31, 4, 2, 64), (1 << 31, 1, 1, 1, 64, 4, 2, 64)):
        assert size(*bad, ops.Q8_0) == 0, bad
