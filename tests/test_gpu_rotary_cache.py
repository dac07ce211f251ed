"""Rotary positions and the paged cache against 64 bits; what an 8-bit cache holds is exact."""
import math

import pytest
import torch

from sensenova_u1_amd import PagedKVCache, RotaryTable, ops, rotary

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu


def _values(gen, tokens, heads, dim):
    return torch.randn((tokens, heads, dim), generator=gen).to(torch.bfloat16)


def _close(got, want, table):
    """Cosine and sine are rounded to fp32 (and so are the two products and their sum), the result to bf16: 4 e (|x| + |y|) m, with |x|, |y| of a
    head at most its largest value, and half a bf16 step of the result."""
    want = want.double()
    size = want.abs().amax(-1, keepdim=True)
    most = 1.01 * (2.0 ** -8 * want.abs() + 8 * 2.0 ** -24 * max(1.0, table.magnitude) * size) + 1e-40
    off = (got.double().cpu() - want).abs()
    assert bool((off <= most).all()), float((off / most).max())


@pytest.mark.parametrize("tokens", [1, 2, 3, 17, 64, 300])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_heads,k_heads,dim,pairs", [(32, 8, 128, 64), (4, 1, 64, 16), (3, 3, 96, 24), (5, 2, 80, 20), (2, 1, 256, 128), (7, 0, 8, 4), (1, 1, 8, 1),
                                                        (2, 2, 128, 33), (2, 1, 136, 68), (1, 1, 1024, 512)])
def test_rotary(dev, tokens, interleaved, q_heads, k_heads, dim, pairs):
    gen = torch.Generator().manual_seed(tokens + dim)
    q, k = _values(gen, tokens, q_heads, dim), _values(gen, tokens, k_heads, dim) if k_heads else None
    positions = torch.randint(0, 5000, (tokens,), generator=gen)
    turns = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)) / (2 * math.pi)
    table = RotaryTable(turns.to(dev), interleaved, 1.25)
    q2, k2 = rotary(q.to(dev), k.to(dev) if k_heads else None, positions.to(dev), table)
    _close(q2, ao.turned(q, positions, turns, interleaved, 1.25), table)
    assert torch.equal(q2[..., 2 * pairs:].cpu(), q[..., 2 * pairs:])
    if k_heads:
        _close(k2, ao.turned(k, positions, turns, interleaved, 1.25), table)
    # in place, and in the memory of a stacked projection
    both = torch.cat([q] + ([k] if k_heads else []), 1).to(dev)
    a, b = both[:, :q_heads], both[:, q_heads:] if k_heads else None
    c, d = rotary(a, b, positions.to(dev), table, inplace=True)
    assert c.data_ptr() == a.data_ptr() and torch.equal(a, q2) and (not k_heads or (torch.equal(b, k2) and d.data_ptr() == b.data_ptr()))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_rows_that_start_anywhere(dev, interleaved):
    gen = torch.Generator().manual_seed(1)
    q, k = _values(gen, 40, 4, 64).to(dev), _values(gen, 40, 2, 64).to(dev)
    positions = torch.arange(40, device=dev) * 1000
    table = RotaryTable.for_model(32, 10000.0, interleaved=interleaved, device=dev)
    want = rotary(q, k, positions, table)
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device=dev)[1:].view(x.shape).copy_(x) for x in (q, k)]
    flipped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
    apart = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]
    wide = [torch.randn((40, x.shape[1], 67), device=dev).to(x.dtype)[..., 3:] for x in (q, k)]
    for w, x in zip(wide, (q, k)):
        w.copy_(x)
    for case in (odd, flipped, apart, wide):
        got = rotary(*case, positions, table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for case in (odd, flipped, wide):
        rotary(*case, positions, table, inplace=True)
        assert torch.equal(case[0], want[0]) and torch.equal(case[1], want[1])


def test_rotary_of_far_and_negative_positions(dev):
    gen = torch.Generator().manual_seed(2)
    positions = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 + 7, -(2 ** 33), 10 ** 9, 131071])
    q = _values(gen, len(positions), 3, 128)
    table = RotaryTable.for_model(128, 1e6, device=dev)
    _close(rotary(q.to(dev), None, positions.to(dev), table)[0], ao.turned(q, positions, table.turns), table)


def test_rotary_table_settings(dev):
    plain = RotaryTable.for_model(64, 10000.0, device=dev)
    want = torch.tensor([10000.0 ** (-2 * i / 64) / (2 * math.pi) for i in range(32)], dtype=torch.float64)
    assert torch.allclose(plain.turns.cpu(), want, rtol=1e-14, atol=0) and plain.magnitude == 1.0
    linear = RotaryTable.for_model(64, 10000.0, scaling="linear", factor=4.0, device=dev)
    assert torch.allclose(linear.turns.cpu(), want / 4, rtol=1e-14, atol=0)
    yarn = RotaryTable.for_model(64, 10000.0, scaling="yarn", factor=8.0, original_context=4096, device=dev)
    assert yarn.magnitude == pytest.approx(0.1 * math.log(8) + 1)
    ratio = (yarn.turns.cpu() / want).tolist()
    rounds = (want * 4096).tolist()
    assert all(r == pytest.approx(1.0) for r, n in zip(ratio, rounds) if n > 40) and all(r == pytest.approx(1 / 8) for r, n in zip(ratio, rounds) if n < 0.7)
    assert all(a >= b - 1e-12 for a, b in zip(ratio, ratio[1:]))


def _cache(dev, pages, heads, page, dim, qt):
    cache = PagedKVCache.empty(pages, heads, page, dim, qt, dev)
    for t in (cache.k, cache.v):
        t.fill_(99)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(7)
    return cache


def _held(cache, name, slots):
    """(whole numbers or values, scales) at slots, as the documented layout says."""
    page = cache.page_size
    s = slots.to(cache.k.device)
    x = getattr(cache, name)[s // page, :, s % page].cpu()
    scale = getattr(cache, name + "_scale")
    return x, scale[s // page, :, :, s % page].cpu() if scale is not None else None


@pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])
@pytest.mark.parametrize("tokens", [1, 5, 64, 333])
@pytest.mark.parametrize("heads,page,dim", [(8, 16, 128), (1, 64, 64), (3, 32, 96), (5, 16, 32), (2, 128, 256), (7, 16, 160)])
def test_cache_write_and_read(dev, qt, tokens, heads, page, dim):
    gen = torch.Generator().manual_seed(tokens + dim)
    k, v = _values(gen, tokens, heads, dim), _values(gen, tokens, heads, dim) * 0.01
    v = v.to(torch.bfloat16)
    pages = -(-tokens // page) + 2
    cache = _cache(dev, pages, heads, page, dim, qt)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    cache.write(k.to(dev), v.to(dev), slots.to(dev))
    got = cache.read(slots.to(dev))
    for name, x, y in (("k", k, got[0]), ("v", v, got[1])):
        held, scale = _held(cache, name, slots)
        if qt == ops.Q8_0:
            q, s, value = ao.quantised(x)
            assert torch.equal(held.double(), q) and torch.equal(scale.double(), s)
            assert torch.equal(y.cpu(), value.float().to(torch.bfloat16))
        else:
            assert torch.equal(held, x) and torch.equal(y.cpu(), x)
    # every other slot is as it was
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    rest = rest.nonzero().flatten()
    held, scale = _held(cache, "k", rest)
    assert bool((held == 99).all()) and (scale is None or bool((scale == 7).all()))


@pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])
def test_slots_outside_the_cache_are_passed_over_and_read_as_zeros(dev, qt):
    gen = torch.Generator().manual_seed(3)
    k, v = _values(gen, 6, 2, 64).to(dev), _values(gen, 6, 2, 64).to(dev)
    cache = _cache(dev, 2, 2, 16, 64, qt)
    slots = torch.tensor([-1, 3, 32, -(2 ** 40), 2 ** 40, 31], device=dev)
    cache.write(k, v, slots)
    a, b = cache.read(slots)
    inside = [1, 5]
    outside = [0, 2, 3, 4]
    assert bool((a[outside] == 0).all()) and bool((b[outside] == 0).all())
    again = PagedKVCache.empty(2, 2, 16, 64, qt, dev)
    again.write(k[inside], v[inside], slots[inside])
    assert torch.equal(again.read(slots[inside])[0], a[inside])
    rest = torch.tensor([s for s in range(32) if s not in (3, 31)])
    assert bool((_held(cache, "v", rest)[0] == 99).all())


def test_8_bit_runs_at_their_ends(dev):
    """Zeros, ties, the smallest scales, saturation, infinities, NaN: run by run."""
    inf, nan = float("inf"), float("nan")
    runs = torch.zeros((12, 32), dtype=torch.float64)
    runs[1, :5] = torch.tensor([127.0, 0.5, 1.5, -2.5, -0.5])            # scale 1: ties go to the even number
    runs[2] = torch.linspace(-3, 3, 32)
    runs[3, :3] = torch.tensor([1e-6, -1e-6, 3e-7])                      # a scale below fp16's normal numbers
    runs[4, :3] = torch.tensor([1e-9, -1e-9, 0.0])                       # a scale of zero: all zero
    runs[5, :3] = torch.tensor([65024.0, -65024.0, 600.0])
    runs[6, :3] = torch.tensor([1e30, -1e6, 600.0])                      # saturates
    runs[7, :3] = torch.tensor([inf, -inf, 1.0])
    runs[8, 7] = nan
    runs[9, 31], runs[9, 0] = nan, inf
    runs[10, 30] = -127.0
    runs[11] = 2.0 ** -130
    x = runs.to(torch.bfloat16).view(3, 2, 64)
    cache = _cache(dev, 1, 2, 16, 64, ops.Q8_0)
    cache.write(x.to(dev), x.to(dev), torch.arange(3, device=dev))
    q, s, value = ao.quantised(x)
    held, scale = _held(cache, "k", torch.arange(3))
    assert torch.equal(held.double(), q) and torch.equal(scale.double().nan_to_num(-1.0), s.nan_to_num(-1.0))
    got = cache.read(torch.arange(3, device=dev))[1].cpu()
    assert torch.equal(got.nan_to_num(-1.0), value.float().to(torch.bfloat16).nan_to_num(-1.0))
    assert bool(got.view(12, 32)[8].isnan().all()) and bool(got.view(12, 32)[9].isnan().all()) and not bool(got.view(12, 32)[:8].isnan().any())


@pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])
@pytest.mark.parametrize("tokens", [1, 24, 131])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_heads,heads,dim,pairs", [(32, 8, 128, 64), (6, 2, 64, 16), (3, 3, 96, 24), (4, 1, 96, 48), (2, 2, 256, 128), (3, 1, 160, 33)])
def test_write_rotary_is_rotary_then_write(dev, qt, tokens, interleaved, q_heads, heads, dim, pairs):
    gen = torch.Generator().manual_seed(tokens)
    qkv = torch.cat([_values(gen, tokens, h, dim) for h in (q_heads, heads, heads)], 1).to(dev)
    q, k, v = qkv.split([q_heads, heads, heads], 1)
    positions = torch.randint(0, 10 ** 6, (tokens,), generator=gen).to(dev)
    turns = 5000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs) / (2 * math.pi)
    table = RotaryTable(turns.to(dev), interleaved)
    slots = torch.randperm(160, generator=gen)[:tokens].to(dev)
    one, two = _cache(dev, 10, heads, 16, dim, qt), _cache(dev, 10, heads, 16, dim, qt)
    q1, k1 = rotary(q, k, positions, table)
    one.write(k1, v, slots)
    q2 = two.write_rotary(q, k, v, positions, table, slots)
    assert torch.equal(q1, q2)
    for a, b in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        assert a is None or torch.equal(a, b)
    before = k.clone()
    q3 = two.write_rotary(q, k, v, positions, table, slots, inplace=True)
    assert q3.data_ptr() == q.data_ptr() and torch.equal(q, q1) and torch.equal(k, before) and torch.equal(one.k, two.k)
    # rows that start anywhere
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device=dev)[1:].view(x.shape).copy_(x) for x in (q1, k, v)]
    three = _cache(dev, 10, heads, 16, dim, qt)
    three.write_rotary(odd[0], odd[1], odd[2], positions, table, slots)
    assert torch.equal(one.k, three.k) and torch.equal(one.v, three.v)
