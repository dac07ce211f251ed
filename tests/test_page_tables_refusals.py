"""What the entry points of the page tables refuse, before anything touches a device (so this runs on a CPU host)."""
import ctypes

import pytest
import torch

from sensenova_u1_amd import PageTables, ops
from sensenova_u1_amd.page_tables import _TABLES

E_SHAPE, E_NULL, E_ALIGN = -2, -3, -4
_BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(_BUF) + 63) // 64 * 64


def _tables(pages=P, lens=P, held=P, free=P, cursor=P, sequences=4, width=4, ring=8, page=16):
    return _TABLES.pack(pages or 0, lens or 0, held or 0, free or 0, cursor or 0, sequences, width, ring, page)


def _append(tables=_tables(), added=P, tokens=4, ends=P, lens=P, cursor=P, positions=P, slots=P, missing=P, ws=None, nbytes=0):
    return ops.load_library().sngguf_page_append(tables, added, tokens, ends, lens, cursor, positions, slots, missing, ws, nbytes, None)


@pytest.mark.parametrize("bad,code", [(dict(sequences=-1), E_SHAPE), (dict(sequences=1 << 24), E_SHAPE), (dict(width=0), E_SHAPE), (dict(width=1 << 27), E_SHAPE), (dict(ring=0), E_SHAPE),
                                      (dict(ring=1 << 31), E_SHAPE), (dict(page=8), E_SHAPE), (dict(page=24), E_SHAPE), (dict(page=8192), E_SHAPE), (dict(pages=None), E_NULL),
                                      (dict(lens=None), E_NULL), (dict(free=None), E_NULL), (dict(cursor=None), E_NULL), (dict(pages=P + 2), E_ALIGN), (dict(cursor=P + 4), E_ALIGN),
                                      (dict(held=P + 1), E_ALIGN)])
def test_tables(bad, code):
    lib = ops.load_library()
    t = _tables(**bad)
    assert _append(tables=t) == code and lib.sngguf_page_release(t, P, None) == code and lib.sngguf_page_fork(t, P, P, None) == code


def test_calls():
    lib = ops.load_library()
    t = _tables()
    assert _append(tables=None) == E_NULL and lib.sngguf_page_release(None, P, None) == E_NULL and lib.sngguf_page_fork(None, P, P, None) == E_NULL
    for bad in (dict(added=None), dict(ends=None), dict(lens=None), dict(cursor=None), dict(positions=None), dict(slots=None), dict(missing=None), dict(tokens=4097)):
        assert _append(**bad) == E_NULL, bad
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(tokens=4097, ws=P, nbytes=63)):
        assert _append(**bad) == E_SHAPE, bad
    for bad in (dict(added=P + 2), dict(positions=P + 4), dict(cursor=P + 4), dict(tokens=4097, ws=P + 8, nbytes=64)):
        assert _append(**bad) == E_ALIGN, bad
    assert lib.sngguf_page_release(t, None, None) == E_NULL
    assert lib.sngguf_page_fork(t, None, P, None) == E_NULL and lib.sngguf_page_fork(_tables(held=None), P, P, None) == E_NULL
    none = _tables(sequences=0, pages=None, lens=None, held=None, free=None, cursor=None)
    assert _append(tables=none, added=None) == 0 and lib.sngguf_page_release(none, None, None) == 0 and lib.sngguf_page_fork(none, None, None, None) == 0
    for sequences, tokens, nbytes in ((1024, 4096, 0), (1025, 1, 1025 * 16), (4, 4097, 64), (0, 9000, 0), (-1, 9000, 0), (4, -1, 0)):
        assert lib.sngguf_page_append_workspace_bytes(sequences, tokens) == nbytes


def test_memory_that_is_shared():
    lib = ops.load_library()
    # arrays 256 bytes apart; each moved into another in turn (a ring of 8, 4 sequences of 4 pages, 4 rows)
    at = {name: P + 256 * i for i, name in enumerate(("pages", "lens", "held", "free", "cursor", "added", "ends", "positions", "slots", "missing"))}
    size = dict(pages=64, lens=16, held=16, free=32, cursor=16, added=16, ends=20, positions=32, slots=32, missing=4)

    def tables(at):
        return _tables(**{n: at[n] for n in ("pages", "lens", "held", "free", "cursor")})

    def append(at):
        return _append(tables(at), **{n: at[n] for n in ("added", "ends", "lens", "cursor", "positions", "slots", "missing")})

    arrays = ("pages", "lens", "held", "free", "cursor")
    for x in arrays:
        for y in arrays:
            if x != y:
                bad = {**at, x: at[y] + size[y] // 8 * 8 - 8}
                assert append(bad) == E_SHAPE and lib.sngguf_page_release(tables(bad), at["added"], None) == E_SHAPE, (x, y)
                assert lib.sngguf_page_fork(tables(bad), at["added"], at["ends"], None) == E_SHAPE, (x, y)
    for y in ("pages", "lens", "cursor", "ends", "positions", "slots", "missing"):
        assert append({**at, "added": at[y] + size[y] - 4}) == E_SHAPE, y
    for y in ("lens", "held", "free", "cursor"):
        assert lib.sngguf_page_release(tables(at), at[y] + size[y] - 1, None) == E_SHAPE, y
    for y in ("pages", "lens", "held"):
        for of in ((at[y] + size[y] - 4, at["ends"]), (at["ends"], at[y] - 12)):
            assert lib.sngguf_page_fork(tables(at), *of, None) == E_SHAPE, y


@pytest.mark.parametrize("tokens,two", [(4, False), (4, True)])
def test_outputs_that_are_shared(tokens, two):
    # arrays 64 KB apart, outputs not in place; with 1025 sequences a workspace as well
    n = 1025 if two else 4
    names = ("pages", "lens", "held", "free", "cursor", "added", "lens_out", "cursor_out", "ends", "missing", "positions", "slots", "workspace")
    room = ctypes.create_string_buffer(14 << 16)
    at = {name: (ctypes.addressof(room) + 63) // 64 * 64 + (i << 16) for i, name in enumerate(names)}
    size = dict(pages=16 * n, lens=4 * n, held=4 * n, free=32, cursor=16, added=4 * n, lens_out=4 * n, cursor_out=16, ends=4 * n + 4, missing=4, positions=8 * tokens, slots=8 * tokens, workspace=16 * n)
    written = names[6:] if two else names[6:-1]

    def append(at):
        return _append(_tables(sequences=n, **{x: at[x] for x in names[:5]}), at["added"], tokens, at["ends"], at["lens_out"], at["cursor_out"], at["positions"], at["slots"], at["missing"],
                       at["workspace"], 16 * n if two else 0)

    for x in written:
        for y in names[:5] + written:
            if x == y:
                continue
            for offset in {0, max(0, size[y] // 16 * 16 - 16), (size[y] - 1) // 8 * 8}:
                if (offset == 0 and (x, y) in (("lens_out", "lens"), ("cursor_out", "cursor"))) or (x == "workspace" and offset % 16):
                    continue
                assert append({**at, x: at[y] + offset}) == E_SHAPE, (x, y, offset)
    for x in ("lens", "cursor"):
        assert append({**at, x + "_out": at[x], "ends": at[x]}) == E_SHAPE


def test_host_tensors():
    for call in (lambda: PageTables.empty(4, 4, 8, 16, device="cpu"), lambda: PageTables.empty(-1, 4, 8, 16, device="cpu"), lambda: PageTables.empty(4, 0, 8, 16, device="cpu"),
                 lambda: PageTables.empty(4, 4, 0, 16, device="cpu")):
        with pytest.raises(ops.SnGgufError):
            call()


def test_the_packed_structure_is_that_of_the_header():
    class Tables(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ("pages", "lens", "held", "free", "cursor")] + [(n, ctypes.c_int64) for n in ("sequences", "width", "ring", "page_size")]

    assert bytes(Tables(1, 2, 3, 4, 5, 6, 7, 8, 9)) == _TABLES.pack(1, 2, 3, 4, 5, 6, 7, 8, 9) and ctypes.sizeof(Tables) == _TABLES.size
