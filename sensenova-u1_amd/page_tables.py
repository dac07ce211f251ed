"""The tables of many sequences over a paged cache, kept and filled on the device: where a step's new tokens lie, their positions and
slots, and the pages of each sequence.  The reference grows one contiguous cache a request (``past_key_values.update``,
``modeling_qwen3.py:483-486,668-671``); a program that serves many requests from one ``PagedKVCache`` needs these at every step.

Nothing here synchronises or reads a length on the host, so a captured step replays with other lengths::

    tables = PageTables.empty(sequences=64, width=256, pages=4096, page_size=64)
    step = tables.append(new, tokens)                    # new: int32 [sequences], how many tokens each gets
    q = cache.write_rotary(q, k, v, step.positions, table, step.slots)
    out = paged_attention(q, cache, tables.pages, step.lens, step.ends)
    tables.release(done)                                 # their pages are free again
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional

import torch

from . import ops
from .attention import _field, _launch, _launch_with_workspace, _numbers, _same_device
from .ops import SnGgufError


# sngguf_page_tables as bytes: pages, lens, held, free, cursor, sequences, width, ring, page_size
_TABLES = struct.Struct("5P4q")


class PageStep(NamedTuple):
    """What a step of many sequences needs: ``ends`` int32 [sequences + 1], where each one's rows start and end; ``lens`` int32 [sequences],
    its tokens behind the step; ``positions`` and ``slots`` int64 [tokens] of each row (0 and -1 behind the last); ``missing`` int32 [1], new tokens
    that found no page.  In place, ``lens`` and ``cursor`` are the tables' own tensors, which the next step changes."""

    ends: torch.Tensor
    lens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    cursor: torch.Tensor
    missing: torch.Tensor


@functools.lru_cache(1024)
def _workspace(sequences: int, tokens: int) -> int:
    return ops.load_library().sngguf_page_append_workspace_bytes(sequences, tokens)


class PageTables:
    """Pages and lengths of ``sequences`` sequences, and the pages that are free.

    ``pages``: int32 [sequences][width], the pages of each sequence in order.  ``lens``: int32 [sequences].  ``free``: int32 [ring], page
    numbers in a ring of at least as many places as there are pages; ``cursor``: int64 [2], how many have been taken from it and given to
    it so far (the c-th lies at place c mod ring, so those from ``cursor[0]`` up to ``cursor[1]`` are there).  ``held``: int32 [sequences], leading pages of a row that
    belong to another sequence (``fork``), None where none do.  No two of them share memory, nor with what a call is given.  ``PageTables.empty`` makes them; the constructor takes tensors that are there.  Calls
    change them in place, on the current stream.  They can be written into, not replaced."""

    __slots__ = ("_pages", "_lens", "_free", "_cursor", "_held", "_page_size", "_tables", "_index", "_sequences", "_lens_at", "_cursor_at", "_memory")
    pages, lens, free, cursor, held, page_size = map(_field, ("pages", "lens", "free", "cursor", "held", "page_size"))

    def __init__(self, pages: torch.Tensor, lens: torch.Tensor, free: torch.Tensor, cursor: torch.Tensor, page_size: int, held: Optional[torch.Tensor] = None) -> None:
        if not pages.is_cuda:
            raise SnGgufError(f"sn_gguf ops run on a HIP device only, got page tables on '{pages.device}'; there is no CPU implementation")
        shape = pages.shape
        if pages.dtype != torch.int32 or len(shape) != 2 or not pages.is_contiguous() or shape[1] < 1:
            raise SnGgufError(f"PageTables: pages must be contiguous int32 [sequences][width], got {pages.dtype} {tuple(shape)}")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise SnGgufError(f"PageTables: pages of 16 .. 4096 tokens (a power of two) are needed, got {page_size}")
        sequences, width = shape
        if width * page_size > (1 << 31) - 65536 or sequences >= 1 << 24:
            raise SnGgufError(f"PageTables: {sequences} sequences of {width} pages of {page_size} tokens are too many")
        for name, x, dtype, count in (("lens", lens, torch.int32, sequences), ("free", free, torch.int32, None), ("cursor", cursor, torch.int64, 2), ("held", held, torch.int32, sequences)):
            if x is not None and _numbers(x, dtype, count, "PageTables", name) is not x:
                raise SnGgufError(f"PageTables: {name} must be contiguous")
        ring = free.numel()
        if not 1 <= ring < 1 << 31:
            raise SnGgufError(f"PageTables: a ring of {ring} pages")
        self._index, self._sequences = pages.get_device(), sequences
        _same_device("PageTables", self._index, lens, free, cursor, held)
        self._pages, self._lens, self._free, self._cursor, self._held, self._page_size = pages, lens, free, cursor, held, int(page_size)
        self._memory = pages.untyped_storage(), lens.untyped_storage(), free.untyped_storage(), cursor.untyped_storage(), None if held is None else held.untyped_storage()
        self._lens_at, self._cursor_at = lens.data_ptr(), cursor.data_ptr()
        self._tables = _TABLES.pack(pages.data_ptr(), self._lens_at, 0 if held is None else held.data_ptr(), free.data_ptr(), self._cursor_at, sequences, width, ring,
                                    self._page_size)

    def __reduce__(self):               # (a copy has the addresses of its own tensors)
        return PageTables, (self._pages, self._lens, self._free, self._cursor, self._page_size, self._held)

    @classmethod
    def empty(cls, sequences: int, width: int, pages: int, page_size: int, device="cuda") -> "PageTables":
        """Tables of ``sequences`` sequences without tokens, of up to ``width`` pages each, with ``pages`` free pages numbered from 0."""
        if sequences < 0 or width < 1 or pages < 1:
            raise SnGgufError(f"PageTables: {sequences} sequences of {width} of {pages} pages")
        table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        lens, held = torch.zeros((2, sequences), dtype=torch.int32, device=device).unbind()
        return cls(table, lens, torch.arange(pages, dtype=torch.int32, device=device), torch.tensor([0, pages], dtype=torch.int64, device=device), page_size, held)

    def append(self, new: torch.Tensor, tokens: int, inplace: bool = True) -> PageStep:
        """A step in which sequence i gets ``new[i]`` tokens (int32 [sequences], 0 among them), packed one sequence after the other into
        ``tokens`` rows: as many as the program's tensors have, the sum of ``new`` or more (rows behind the last are padding; new tokens behind the last row are none).

        Sequences that outgrow their pages get free ones, in order.  A token for which there is none, or whose sequence's row of pages is
        full, has slot -1 and does not count in ``lens``; ``missing`` says how many there are.  Not ``inplace``, lengths and cursor stay as they
        were, and only ``pages`` is filled in, behind what the lengths reach: the same step again gives the same.  ``tables.lens.copy_(step.lens)`` and
        ``tables.cursor.copy_(step.cursor)`` take such a step over."""
        what = "PageTables.append"
        sequences = self._sequences
        new = _numbers(new, torch.int32, sequences, what, "new")
        _same_device(what, self._index, new)
        if not 0 <= tokens < 1 << 31:
            raise SnGgufError(f"{what}: {tokens} rows")
        # (two allocations, each cut in one call)
        positions, slots, cursor = self._cursor.new_empty(2 * tokens + 2).split((tokens, tokens, 2))
        ends, lens, missing = new.new_empty(2 * sequences + 2).split((sequences + 1, sequences, 1))
        if inplace:
            lens, cursor, lens_at, cursor_at = self._lens, self._cursor, self._lens_at, self._cursor_at
        else:
            lens_at, cursor_at = lens.data_ptr(), cursor.data_ptr()
        if sequences:
            _launch_with_workspace(self._index, _workspace(sequences, tokens), "sngguf_page_append", self._tables, new.data_ptr(), tokens, ends.data_ptr(), lens_at, cursor_at,
                                   positions.data_ptr(), slots.data_ptr(), missing.data_ptr())
        else:
            for x in (ends, missing, positions):
                x.zero_()
            slots.fill_(-1)
            if not inplace:
                cursor.copy_(self._cursor)
        return PageStep(ends, lens, positions, slots, cursor, missing)

    def release(self, done: torch.Tensor) -> None:
        """Sequences with ``done`` (bool or uint8 [sequences]) end: the pages of their own are free again, their lengths 0.  One whose pages others
        hold (``fork``) is released behind them."""
        what = "PageTables.release"
        if done.dtype not in (torch.bool, torch.uint8):
            raise SnGgufError(f"{what}: done must be bool or uint8, got {done.dtype}")
        done = _numbers(done, done.dtype, self._sequences, what, "done")
        _same_device(what, self._index, done)
        if self._sequences:
            _launch(self._index, "sngguf_page_release", self._tables, done.data_ptr())

    def fork(self, parent: torch.Tensor, common: torch.Tensor) -> None:
        """Sequence i with ``parent[i]`` >= 0 (int32 [sequences], -1: none) starts with that one's first ``common[i]`` tokens, rounded down to whole pages:
        it holds their pages, and the parent owns them.  Nothing happens to a sequence that has tokens, or whose parent is no sequence or one that
        has a parent in the same call.  What ``shared_prefix_attention`` reads once for all of them."""
        what = "PageTables.fork"
        sequences = self._sequences
        parent, common = _numbers(parent, torch.int32, sequences, what, "parent"), _numbers(common, torch.int32, sequences, what, "common")
        _same_device(what, self._index, parent, common)
        if self._held is None:
            raise SnGgufError(f"{what}: these tables have no record of pages held (`held`)")
        if sequences:
            _launch(self._index, "sngguf_page_fork", self._tables, parent.data_ptr(), common.data_ptr())
