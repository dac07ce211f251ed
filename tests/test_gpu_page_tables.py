"""The tables of many sequences against a program on the host: every number is equal."""
import copy
import pickle
import random

import pytest
import torch

from sensenova_u1_amd import PageTables, ops

from .page_oracle import Tables

pytestmark = pytest.mark.gpu


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _same(tables, oracle):
    assert tables.lens.tolist() == oracle.lens and tables.cursor.tolist() == [oracle.taken, oracle.given] and tables.free.tolist() == oracle.free
    assert tables.held is None or tables.held.tolist() == oracle.held
    rows = tables.pages.tolist()
    for i, row in enumerate(rows):
        assert row[:oracle.has(i)] == oracle.rows[i][:oracle.has(i)], i


def _step(tables, oracle, new, tokens, dev, **kw):
    got = tables.append(_ints(new, dev), tokens, **kw)
    want = oracle.append(new, tokens)
    for name, x in want.items():
        mine = getattr(got, name)
        assert mine.dtype == x.dtype and torch.equal(mine.cpu(), x), (name, mine.tolist()[:50], x.tolist()[:50])
    return got


@pytest.mark.parametrize("sequences,width,pages,page,most", [(1, 4, 4, 16, 30), (3, 8, 20, 16, 9), (24, 40, 300, 32, 60), (64, 9, 200, 16, 40), (200, 20, 2500, 16, 3), (7, 3, 9, 64, 200)])
def test_a_service(dev, sequences, width, pages, page, most):
    rng = random.Random(sequences)
    tables, oracle = PageTables.empty(sequences, width, pages, page, dev), Tables(sequences, width, pages, page)
    for turn in range(12):
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(sequences)]
        _step(tables, oracle, new, sum(new) + rng.choice([0, 0, 5]), dev)
        done = [rng.random() < 0.3 for _ in range(sequences)]
        if turn % 2:
            # a child and its parent end together: the parent's pages are its own
            for i in range(sequences):
                if oracle.held[i]:
                    done[i] = True
            tables.release(torch.tensor(done, device=dev))
            oracle.release(done)
        else:
            free = [i for i in range(sequences) if not oracle.lens[i]]
            parent, common = [-1] * sequences, [rng.randint(-3, width * page) for _ in range(sequences)]
            for i in free:
                parent[i] = rng.choice([-1, rng.randrange(-2, sequences + 2)])
            tables.fork(_ints(parent, dev), _ints(common, dev))
            oracle.fork(parent, common)
        _same(tables, oracle)


def test_all_lengths_of_one_launch_and_two(dev):
    # the border of the two forms, in sequences and in rows, and many rows of few sequences
    for sequences, new, tokens in ((1024, 1, 1024), (1025, 1, 1025), (1024, 4, 4096), (1024, 4, 4097), (5000, 2, 10000), (2, 20000, 40003), (4097, 1, 4097), (4096, 1, 4200)):
        rng = random.Random(tokens)
        page = 16
        width = -(-(40 + 2 * new) // page)
        pages = sequences * width
        tables, oracle = PageTables.empty(sequences, width, pages, page, dev), Tables(sequences, width, pages, page)
        first = [rng.randint(0, 30) for _ in range(sequences)]
        _step(tables, oracle, first, sum(first), dev)
        _step(tables, oracle, [rng.choice([0, new, new]) for _ in range(sequences)], tokens, dev)
        _same(tables, oracle)


def test_too_few_pages_and_full_rows(dev):
    tables, oracle = PageTables.empty(5, 3, 6, 16, dev), Tables(5, 3, 6, 16)
    assert _step(tables, oracle, [20, 0, 33, 16, 17], 86, dev).missing.item() > 0     # 2 + 3 + 1 pages, then none
    _same(tables, oracle)
    _step(tables, oracle, [12, 5, 100, 1, 0], 118, dev)                                # room in a page that is there; a row that is full
    _same(tables, oracle)
    done = [False, False, True, False, False]
    tables.release(torch.tensor(done, device=dev))
    oracle.release(done)
    _step(tables, oracle, [0, 17, 0, 0, 17], 34, dev)
    _same(tables, oracle)


def test_more_new_tokens_than_rows_and_negative_ones(dev):
    tables, oracle = PageTables.empty(4, 4, 16, 16, dev), Tables(4, 4, 16, 16)
    _step(tables, oracle, [5, -7, 10, 20], 11, dev)
    _same(tables, oracle)
    _step(tables, oracle, [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 1], 70, dev)
    _same(tables, oracle)
    _step(tables, oracle, [1, 1, 1, 1], 0, dev)
    _same(tables, oracle)


def test_not_in_place(dev):
    tables, oracle = PageTables.empty(6, 10, 40, 16, dev), Tables(6, 10, 40, 16)
    _step(tables, oracle, [3, 40, 0, 16, 17, 1], 77, dev)
    before = tables.lens.clone(), tables.cursor.clone()
    new = _ints([30, 1, 5, 0, 16, 100], dev)
    one = tables.append(new, 160, inplace=False)
    assert torch.equal(tables.lens, before[0]) and torch.equal(tables.cursor, before[1])
    pages = tables.pages.clone()
    two = tables.append(new, 160, inplace=False)
    assert all(torch.equal(a, b) for a, b in zip(one, two)) and torch.equal(pages, tables.pages)
    three = tables.append(new, 160)
    assert all(torch.equal(a, b) for a, b in zip(one, three)) and three.lens is tables.lens and torch.equal(tables.cursor, one.cursor)


def test_a_ring_that_has_gone_round_many_times(dev):
    page, pages = 16, 11
    tables, oracle = PageTables.empty(3, 5, pages, page, dev), Tables(3, 5, pages, page)
    far = (1 << 40) // pages * pages
    tables.cursor += far
    oracle.taken, oracle.given = far, far + pages
    rng = random.Random(1)
    for _ in range(40):
        new = [rng.randint(0, 40) for _ in range(3)]
        _step(tables, oracle, new, sum(new), dev)
        done = [rng.random() < 0.6 for _ in range(3)]
        tables.release(torch.tensor(done, dtype=torch.uint8, device=dev))
        oracle.release(done)
        _same(tables, oracle)


def test_numbers_that_are_none_stay_within_the_tensors(dev):
    """Lengths, cursors and pages that no program has: nothing outside the tables is read or written."""
    room = torch.full((3, 8, 4), 77, dtype=torch.int32, device=dev)
    for lens, cursor in (([-5, 10 ** 9, 3, 64, 0, -2 ** 31, 2 ** 31 - 1, 63], [0, 20]), ([0] * 8, [5, 2]), ([0] * 8, [-3, 10 ** 12]), ([0] * 8, [-(2 ** 62), -(2 ** 62) + 4])):
        room.fill_(77)
        ring = torch.full((60,), 77, dtype=torch.int32, device=dev)
        ring[20:40] = torch.arange(20, device=dev, dtype=torch.int32)
        tables = PageTables(room[1], _ints(lens, dev), ring[20:40], torch.tensor(cursor, device=dev), 16, held=_ints([3, -9, 100, 0, 0, 0, 0, 0], dev))
        step = tables.append(_ints([9] * 8, dev), 72)
        assert bool((step.lens >= 0).all()) and bool((step.lens <= 64).all()) and step.ends.tolist() == list(range(0, 73, 9))
        tables.fork(_ints([1, -1, 7, 2 ** 31 - 1, -2 ** 31, 5, 6, 7], dev), _ints([2 ** 31 - 1] * 8, dev))
        tables.release(torch.ones(8, dtype=torch.bool, device=dev))
        assert bool((room[0] == 77).all()) and bool((room[2] == 77).all()) and bool((ring[:20] == 77).all()) and bool((ring[40:] == 77).all())
        assert tables.lens.tolist() == [0] * 8


@pytest.mark.parametrize("tokens", [96, 5000])
def test_captured_steps(dev, tokens):
    sequences, page, pages, width = 16, 16, 150, 12
    tables, oracle = PageTables.empty(sequences, width, pages, page, dev), Tables(sequences, width, pages, page)
    new, done = _ints([0] * sequences, dev), torch.zeros(sequences, dtype=torch.bool, device=dev)
    tables.append(new, tokens)
    tables.release(done)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables.release(done)
        step = tables.append(new, tokens)
    rng = random.Random(2)
    for turn in range(10):
        of, gone = [rng.randint(0, 6) for _ in range(sequences)], [rng.random() < 0.2 for _ in range(sequences)]
        new.copy_(_ints(of, dev))
        done.copy_(torch.tensor(gone))
        graph.replay()
        oracle.release(gone)
        want = oracle.append(of, tokens)
        for name, x in want.items():
            assert torch.equal(getattr(step, name).cpu(), x), (turn, name)
        _same(tables, oracle)
        PageTables.empty(sequences, width, pages, page, dev).append(new, 9000)         # (the program's own eager work between)


def test_no_sequences_and_no_rows(dev):
    tables = PageTables.empty(0, 4, 8, 16, dev)
    step = tables.append(_ints([], dev), 3)
    assert step.ends.tolist() == [0] and step.slots.tolist() == [-1] * 3 and step.positions.tolist() == [0] * 3 and step.missing.tolist() == [0] and step.cursor.tolist() == [0, 8]
    tables.release(torch.zeros(0, dtype=torch.bool, device=dev))
    tables.fork(_ints([], dev), _ints([], dev))


def test_what_is_refused(dev):
    tables = PageTables.empty(4, 4, 8, 16, dev)
    good = dict(pages=tables.pages, lens=tables.lens, free=tables.free, cursor=tables.cursor, page_size=16)
    for bad in (dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(lens=tables.lens[:3]), dict(lens=tables.lens.long()), dict(cursor=tables.cursor.int()), dict(pages=tables.pages.long()),
                dict(pages=tables.pages.T), dict(free=tables.free[:0]), dict(free=tables.free[::2]), dict(held=tables.lens[:2]), dict(lens=torch.zeros((4, 2), dtype=torch.int32, device=dev)[:, 0]),
                dict(lens=tables.lens.cpu())):
        with pytest.raises(ops.SnGgufError):
            PageTables(**{**good, **bad})
    new = _ints([1] * 4, dev)
    for call in (lambda: tables.append(new[:3], 4), lambda: tables.append(new.long(), 4), lambda: tables.append(new, -1), lambda: tables.append(new.cpu(), 4), lambda: tables.release(new),
                 lambda: tables.release(torch.zeros(3, dtype=torch.bool, device=dev)), lambda: tables.fork(new, new[:2]), lambda: PageTables(**good).fork(new, new)):
        with pytest.raises(ops.SnGgufError):
            call()


def test_copies_have_tensors_of_their_own(dev):
    tables, oracle = PageTables.empty(3, 4, 12, 16, dev), Tables(3, 4, 12, 16)
    _step(tables, oracle, [20, 0, 3], 23, dev)
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables))):
        before = [t.clone() for t in (tables.pages, tables.lens, tables.cursor, tables.free)]
        their = copy.deepcopy(oracle)
        _step(other, their, [1, 40, 13], 54, dev)
        other.release(torch.tensor([True, False, False], device=dev))
        their.release([True, False, False])
        _same(other, their)
        assert all(torch.equal(a, b) for a, b in zip(before, (tables.pages, tables.lens, tables.cursor, tables.free)))
    same = copy.copy(tables)
    assert same.lens is tables.lens
    _step(same, oracle, [5, 5, 5], 15, dev)
    _same(tables, oracle)


def test_numbers_in_the_tables_own_memory_are_refused(dev):
    tables = PageTables.empty(4, 4, 8, 16, dev)
    room = torch.zeros(5, dtype=torch.int32, device=dev)
    shifted = PageTables(tables.pages, room[1:], tables.free, tables.cursor, 16, held=tables.held)
    done = tables.lens.view(torch.uint8)[:4]
    for call in (lambda: tables.append(tables.lens, 4), lambda: shifted.append(room[:4], 4), lambda: tables.append(tables.pages[0], 4), lambda: tables.release(done),
                 lambda: tables.fork(tables.held, room[:4]), lambda: PageTables(tables.pages, tables.pages[0], tables.free, tables.cursor, 16).append(room[:4], 4)):
        with pytest.raises(ops.SnGgufError):
            call()
    assert tables.append(tables.lens, 4, inplace=False).missing.item() == 0          # (nothing of it is written)
