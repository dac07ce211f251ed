"""What is made of tensors keeps the memory whose addresses it passes on, whatever becomes of the tensors.  Without a device, host tensors stand in for its:
nothing is launched there."""
import copy
import gc
import weakref

import numpy as np
import pytest
import torch

from sensenova_u1_amd import HeadNorm, PagedKVCache, PageTables, RotaryAxes, RotaryTable, ops, paged_attention, rotary
from sensenova_u1_amd.attention import _NORM


class Standing(torch.Tensor):
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


class StandingParameter(torch.nn.Parameter):
    is_cuda, get_device = Standing.is_cuda, Standing.get_device

    def detach(self):                   # (a parameter's is a plain tensor)
        return torch.Tensor._make_subclass(Standing, super().detach())


def _page_tables(pages, lens, free, cursor, held):
    return PageTables(pages, lens, free, cursor, 16, held)


# how it is made, of which arrays (aligned, as the constructors copy others), and the fields that hold them
MAKERS = {
    "HeadNorm": (HeadNorm, [((64,), "float32"), ((64,), "float32")], lambda x: x.weights),
    "RotaryTable": (RotaryTable, [((32,), "float64")], lambda x: (x.turns,)),
    "RotaryAxes": (RotaryAxes, [((32,), "float64"), ((32,), "int32")], lambda x: (x.turns, x.axis)),
    "PageTables": (_page_tables, [((4, 3), "int32"), ((4,), "int32"), ((12,), "int32"), ((2,), "int64"), ((4,), "int32")], lambda x: (x.pages, x.lens, x.free, x.cursor, x.held)),
    "PagedKVCache": (PagedKVCache, [((2, 1, 16, 64), "int8")] * 2 + [((2, 1, 2, 16), "float16")] * 2, lambda x: (x.k, x.v, x.k_scale, x.v_scale)),
}


def _array(shape, dtype):
    size = int(np.prod(shape)) * np.dtype(dtype).itemsize
    room = np.zeros(size + 64, np.uint8)
    start = -room.ctypes.data % 64
    return room[start:start + size].view(dtype).reshape(shape)


def _made(name, kind):
    make, arrays, fields = MAKERS[name]
    tensors, memory = [], []
    for shape, dtype in arrays:
        a = _array(shape, dtype)
        memory.append(weakref.ref(a))
        tensors.append(torch.Tensor._make_subclass(kind, torch.from_numpy(a)))
    return make(*tensors), tensors, memory, fields


@pytest.mark.parametrize("kind", [Standing, StandingParameter])
@pytest.mark.parametrize("name", MAKERS)
def test_tensors_that_are_given_other_memory(name, kind):
    x, tensors, memory, fields = _made(name, kind)
    alike = copy.copy(x)
    assert all(m() is not None for m in memory)
    for t in (*tensors, *fields(x)):
        t.data = torch.zeros_like(t)
    del tensors, t
    gc.collect()
    assert all(m() is not None for m in memory)
    del x
    gc.collect()
    assert all(m() is not None for m in memory)        # (the copy has the same)
    del alike
    gc.collect()
    assert all(m() is None for m in memory)


def test_a_norm_of_parameters_shows_the_weights_that_it_reads():
    x, tensors, _, _ = _made("HeadNorm", StandingParameter)
    at = [t.data_ptr() for t in tensors]
    for t in tensors:
        t.data = torch.ones_like(t)
    assert [w.data_ptr() for w in x.weights] == at == list(_NORM.unpack(x._norm)[:2]) and [w.data_ptr() for w in copy.copy(x).weights] == at


FIELDS = {"HeadNorm": "weights eps dim", "RotaryTable": "turns interleaved magnitude", "RotaryAxes": "turns axis parts interleaved magnitude",
          "PageTables": "pages lens free cursor held page_size", "PagedKVCache": "k v k_scale v_scale quant_type pages kv_heads page_size dim"}


@pytest.mark.parametrize("name,field", [(name, f) for name, fields in FIELDS.items() for f in fields.split()])
def test_fields_cannot_be_replaced(name, field):
    x = _made(name, Standing)[0]
    held = getattr(x, field)
    setattr(x, field, held)             # (as x.field += 1 does)
    for value in (held.clone() if isinstance(held, torch.Tensor) else "other", None):
        with pytest.raises(ops.SnGgufError, match=f"{name}: {field} cannot be replaced"):
            setattr(x, field, value)
    with pytest.raises(AttributeError):
        delattr(x, field)
    assert getattr(x, field) is held and getattr(copy.copy(x), field) is not None


@pytest.mark.gpu
def test_a_step_that_was_not_in_place_is_taken_over(dev):
    tables, same = (PageTables.empty(3, 4, 12, 16, dev) for _ in range(2))
    for new in ([5, 0, 20], [13, 1, 30], [0, 40, 1]):
        new = torch.tensor(new, dtype=torch.int32, device=dev)
        step, want = tables.append(new, 50, inplace=False), same.append(new, 50)
        with pytest.raises(ops.SnGgufError, match="lens cannot be replaced"):
            tables.lens = step.lens
        tables.lens.copy_(step.lens)
        tables.cursor.copy_(step.cursor)
        assert all(torch.equal(a, b) for a, b in zip(step, want)) and torch.equal(tables.pages, same.pages) and torch.equal(tables.lens, same.lens)


@pytest.mark.gpu
def test_calls_read_what_they_were_made_with(dev):
    gen = torch.Generator().manual_seed(1)
    q, at, slots = torch.randn((3, 2, 64), generator=gen).to(torch.bfloat16).to(dev), torch.arange(3, device=dev), torch.arange(3, device=dev)
    weight = torch.nn.Parameter(torch.linspace(0.5, 2, 64, device=dev), requires_grad=False)
    norm, table, axes = HeadNorm(weight), RotaryTable.for_model(64, device=dev), RotaryAxes.for_model([(64, 0, 1e4)], device=dev)
    cache, tables = PagedKVCache.empty(2, 2, 16, 64, ops.Q8_0, dev), PageTables.empty(3, 2, 6, 16, dev)
    ones = torch.ones(3, dtype=torch.int32, device=dev)

    def results():
        tables.append(ones, 3)
        pages, lens = torch.zeros((3, 1), dtype=torch.int32, device=dev), torch.full((3,), 3, dtype=torch.int32, device=dev)
        one, two = cache.write_rotary(q, q, q, at, table, slots, q_norm=norm, k_norm=norm), rotary(q, None, at[None], axes, q_norm=norm)[0]
        return one, two, *cache.read(slots), paged_attention(q, cache, pages, lens)

    want = results()
    weight.data = torch.full((64,), 3.0, device=dev)
    for t in (norm.weights[0], table.turns, axes.turns, axes.axis, cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.data = torch.full_like(t, 5)
    lens, cursor = tables.lens.view(-1), tables.cursor.view(-1)
    for t in (tables.pages, tables.lens, tables.free, tables.cursor, tables.held):
        t.data = torch.full_like(t, 7)
    torch.cuda.empty_cache()
    room = [torch.full((1 << 16,), 9, dtype=torch.uint8, device=dev) for _ in range(20)]       # (freed memory would be given out again)
    assert all(torch.equal(a, b) for a, b in zip(results(), want)) and len(room) == 20
    assert lens.tolist() == [2, 2, 2] and cursor.tolist() == [3, 6]
