"""Norms of single heads and rotation by several positions, to tensors and into the cache, against 64 bits."""
import copy
import math
import pickle

import pytest
import torch

from sensenova_u1_amd import HeadNorm, PagedKVCache, RotaryAxes, RotaryTable, ops, rotary

from . import attention_oracle as ao
from . import head_oracle as ho

pytestmark = pytest.mark.gpu


def _values(gen, tokens, heads, dim):
    return torch.randn((tokens, heads, dim), generator=gen).to(torch.bfloat16)


def _weights(gen, sizes, kind=torch.bfloat16):
    return [(1 + 0.4 * torch.randn(n, generator=gen)).to(kind) for n in sizes]


def _table(gen, parts, axes):
    pairs = sum(parts) // 2
    turns = torch.cat([10000.0 ** (-torch.arange(n // 2, dtype=torch.float64) / (n // 2)) / (2 * math.pi) for n in parts])
    return turns, torch.randint(0, axes, (pairs,), generator=gen, dtype=torch.int32)


def _close(got, want, most):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= most).all()), float((off / most).max())


SHAPES = [  # q heads, k heads, dim, parts of the rotation, parts of the norm
    (32, 8, 128, (64, 32, 32), (64, 64)), (32, 8, 128, (128,), (128,)), (4, 1, 64, (32, 16, 16), (32, 32)), (3, 3, 96, (48, 24, 24), (96,)), (2, 1, 96, (48, 24, 24), (48, 48)),
    (5, 2, 80, (40,), (80,)), (2, 1, 256, (128, 64, 64), (128, 128)), (7, 0, 8, (2, 2, 2, 2), (8,)), (1, 1, 8, (6,), (8,)), (2, 2, 128, (66,), (8, 24, 32, 64)),
    (2, 1, 136, (16, 34), (64, 72)), (1, 2, 512, (256, 256), (512,)), (3, 1, 512, (512,), (128, 128, 128, 128)), (2, 2, 128, (96, 16), (32, 96)), (40, 8, 64, (64,), ())]


@pytest.mark.parametrize("tokens", [1, 2, 5, 33, 130])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_heads,k_heads,dim,parts,norm", SHAPES)
def test_normed_and_turned(dev, tokens, interleaved, q_heads, k_heads, dim, parts, norm):
    gen = torch.Generator().manual_seed(tokens + dim)
    q, k = _values(gen, tokens, q_heads, dim), _values(gen, tokens, k_heads, dim) if k_heads else None
    turns, axis = _table(gen, parts, 3)
    positions = torch.randint(0, 5000, (3, tokens), generator=gen)
    kind = torch.float32 if tokens % 2 else torch.bfloat16
    qw, kw = _weights(gen, norm, kind), _weights(gen, norm, kind)
    table = RotaryAxes(turns.to(dev), axis.to(dev), parts, interleaved, 1.25)
    norms = dict(q_norm=HeadNorm(*(w.to(dev) for w in qw), eps=1e-5), k_norm=HeadNorm(*(w.to(dev) for w in kw), eps=1e-5)) if norm else {}
    on = positions.to(dev)
    q2, k2 = rotary(q.to(dev), k.to(dev) if k_heads else None, on, table, **norms)
    _close(q2, *ho.head(q, positions, turns, axis, parts, interleaved, 1.25, qw, 1e-5))
    if k_heads:
        _close(k2, *ho.head(k, positions, turns, axis, parts, interleaved, 1.25, kw, 1e-5))
    if not norm:
        assert torch.equal(q2[..., sum(parts):].cpu(), q[..., sum(parts):])
    # one norm alone leaves the other's heads turned only
    if norm and k_heads:
        q3, k3 = rotary(q.to(dev), k.to(dev), on, table, k_norm=norms["k_norm"])
        assert torch.equal(k3, k2)
        _close(q3, *ho.head(q, positions, turns, axis, parts, interleaved, 1.25))
    # in place, and in the memory of a stacked projection
    both = torch.cat([q] + ([k] if k_heads else []), 1).to(dev)
    a, b = both[:, :q_heads], both[:, q_heads:] if k_heads else None
    c, d = rotary(a, b, on, table, inplace=True, **norms)
    assert c.data_ptr() == a.data_ptr() and torch.equal(a, q2) and (not k_heads or (torch.equal(b, k2) and d.data_ptr() == b.data_ptr()))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pairs,dim", [(64, 128), (24, 96), (20, 80), (4, 8), (33, 128)])
def test_a_table_of_one_position_with_norms(dev, interleaved, pairs, dim):
    gen = torch.Generator().manual_seed(pairs)
    q, k, w = _values(gen, 19, 6, dim), _values(gen, 19, 2, dim), _weights(gen, (dim,))
    positions = torch.randint(0, 100000, (19,), generator=gen)
    table = RotaryTable.for_model(2 * pairs, 1e6, interleaved=interleaved, device=dev)
    norm = HeadNorm(w[0].to(dev))
    q2, k2 = rotary(q.to(dev), k.to(dev), positions.to(dev), table, q_norm=norm, k_norm=norm)
    axis = torch.zeros(pairs, dtype=torch.int32)
    _close(q2, *ho.head(q, positions[None], table.turns, axis, (2 * pairs,), interleaved, 1.0, w))
    _close(k2, *ho.head(k, positions[None], table.turns, axis, (2 * pairs,), interleaved, 1.0, w))
    # the same table as one of several axes, all pairs by the first
    same = RotaryAxes(table.turns, axis.to(dev), interleaved=interleaved)
    q3, k3 = rotary(q.to(dev), k.to(dev), torch.stack([positions, -positions]).to(dev), same, q_norm=norm, k_norm=norm)
    assert torch.equal(q3, q2) and torch.equal(k3, k2)
    # keys alone
    none, k4 = rotary(q[:, :0].to(dev), k.to(dev), positions.to(dev), table, q_norm=norm, k_norm=norm)
    assert none.shape == (19, 0, dim) and torch.equal(k4, k2)


def test_one_axis_without_norms_is_the_plain_rotation(dev):
    gen = torch.Generator().manual_seed(3)
    q, k = _values(gen, 50, 32, 128).to(dev), _values(gen, 50, 8, 128).to(dev)
    positions = torch.randint(0, 1 << 20, (50,), generator=gen).to(dev)
    for interleaved in (False, True):
        table = RotaryTable.for_model(128, 1e6, interleaved=interleaved, device=dev)
        axes = RotaryAxes(table.turns, torch.zeros(64, dtype=torch.int32, device=dev), interleaved=interleaved)
        want, got = rotary(q, k, positions, table), rotary(q, k, positions[None], axes)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_table_of_parts(dev):
    table = RotaryAxes.for_model([(64, 0, 5e6), (32, 1, 1e4), (32, 2, 1e4)], device=dev)
    assert table.parts == (64, 32, 32) and table.axis.tolist() == [0] * 32 + [1] * 16 + [2] * 16
    want = [5e6 ** (-i / 32) / (2 * math.pi) for i in range(32)] + 2 * [1e4 ** (-i / 16) / (2 * math.pi) for i in range(16)]
    assert table.turns.tolist() == pytest.approx(want, rel=1e-14)
    # each part as a call of its own on a view
    gen = torch.Generator().manual_seed(4)
    q = _values(gen, 37, 4, 128).to(dev)
    positions = torch.randint(0, 300, (3, 37), generator=gen).to(dev)
    got, _ = rotary(q, None, positions, table)
    start = 0
    for i, (n, base) in enumerate(((64, 5e6), (32, 1e4), (32, 1e4))):
        part = rotary(q[..., start:start + n], None, positions[i], RotaryTable.for_model(n, base, device=dev))[0]
        assert torch.equal(got[..., start:start + n], part)
        start += n


@pytest.mark.parametrize("parts", [(32, 16, 16), (26, 18, 4)])
def test_rows_that_start_anywhere(dev, parts):
    gen = torch.Generator().manual_seed(1)
    q, k = _values(gen, 40, 4, 64).to(dev), _values(gen, 40, 2, 64).to(dev)
    turns, axis = _table(gen, parts, 3)
    table, positions = RotaryAxes(turns.to(dev), axis.to(dev), parts), torch.randint(0, 99, (3, 40), generator=gen).to(dev)
    norms = dict(q_norm=HeadNorm(*(w.to(dev) for w in _weights(gen, (32, 32)))), k_norm=HeadNorm(_weights(gen, (64,))[0].to(dev)))
    want = rotary(q, k, positions, table, **norms)
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device=dev)[1:].view(x.shape).copy_(x) for x in (q, k)]
    flipped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
    apart = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]
    wide = [torch.randn((40, x.shape[1], 67), device=dev).to(x.dtype)[..., 3:] for x in (q, k)]
    for w, x in zip(wide, (q, k)):
        w.copy_(x)
    for case in (odd, flipped, apart, wide):
        got = rotary(*case, positions, table, **norms)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # positions as [tokens][axes] seen from the other side, and rows of more tokens than there are
    for p in (positions.T.contiguous().T, torch.cat([positions, positions], 1)[:, :40]):
        got = rotary(q, k, p, table, **norms)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for case in (odd, flipped, wide):
        rotary(*case, positions, table, inplace=True, **norms)
        assert torch.equal(case[0], want[0]) and torch.equal(case[1], want[1])
    # weights at any address
    room = torch.empty(33, dtype=torch.bfloat16, device=dev)
    w = norms["q_norm"].weights
    shifted = HeadNorm(room[1:].copy_(w[0]), w[1])
    assert torch.equal(rotary(q, None, positions, table, q_norm=HeadNorm(*w))[0], rotary(q, None, positions, table, q_norm=shifted)[0])


def test_far_negative_and_missing_positions(dev):
    gen = torch.Generator().manual_seed(2)
    positions = torch.tensor([[0, 1, -1, 2 ** 20 + 1, 2 ** 31 + 7, -(2 ** 33), 10 ** 9, 131071], [5, 4, 3, 2, 1, 0, -1, -2]])
    q = _values(gen, 8, 3, 128)
    turns, axis = _table(gen, (64, 64), 2)
    axis[:3] = torch.tensor([-5, 2, 100], dtype=torch.int32)       # axes that positions do not have: the nearest
    got, _ = rotary(q.to(dev), None, positions.to(dev), RotaryAxes(turns.to(dev), axis.to(dev), (64, 64)))
    _close(got, *ho.head(q, positions, turns, axis, (64, 64)))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [4, 5, 9])
def test_more_axes(dev, axes, interleaved):
    gen = torch.Generator().manual_seed(axes)
    q, positions = _values(gen, 21, 3, 128), torch.randint(-50, 5000, (axes, 21), generator=gen)
    turns, axis = _table(gen, (64, 32, 32), axes)
    axis[:3] = torch.tensor([-1, axes, axes - 1], dtype=torch.int32)
    table, weights = RotaryAxes(turns.to(dev), axis.to(dev), (64, 32, 32), interleaved), _weights(gen, (128,))
    got, _ = rotary(q.to(dev), None, positions.to(dev), table, q_norm=HeadNorm(weights[0].to(dev)))
    _close(got, *ho.head(q, positions, turns, axis, (64, 32, 32), interleaved, weights=weights))
    # positions of some of many axes, every other token, one axis for all
    many = torch.randint(-50, 5000, (axes, 2 * 21), generator=gen)
    got, _ = rotary(q.to(dev), None, many.to(dev)[:, ::2], table)
    _close(got, *ho.head(q, many[:, ::2], turns, axis, (64, 32, 32), interleaved))
    got, _ = rotary(q.to(dev), None, many[:1, :21].to(dev).expand(axes, 21), table)
    _close(got, *ho.head(q, many[:1, :21].expand(axes, 21), turns, axis, (64, 32, 32), interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
def test_magnitudes(dev, interleaved):
    """Parts of very small and very large elements; squares beyond 32 bits make a part zeros."""
    gen = torch.Generator().manual_seed(3)
    turns, axis = _table(gen, (64,), 1)
    table, weights, at = RotaryAxes(turns.to(dev), axis.to(dev), (64,), interleaved), _weights(gen, (64,)), torch.arange(5)[None]
    norm = HeadNorm(weights[0].to(dev), eps=0.0)
    for size in (1e-19, 1e-12, 1e17):
        q = (_values(gen, 5, 2, 64).float() * size).to(torch.bfloat16)
        _close(rotary(q.to(dev), None, at.to(dev), table, q_norm=norm)[0], *ho.head(q, at, turns, axis, (64,), interleaved, weights=weights, eps=0.0))
    q = torch.full((5, 2, 64), 1e30, dtype=torch.bfloat16)
    assert not rotary(q.to(dev), None, at.to(dev), table, q_norm=norm)[0].any()


@pytest.mark.parametrize("parts", [(64,), (32, 16, 16), (50, 6)])
def test_rows_that_are_not_finite_and_rows_of_zeros(dev, parts):
    gen = torch.Generator().manual_seed(5)
    q = _values(gen, 6, 3, 64)
    q[0, 1, 5] = torch.nan
    q[1, 0, 63] = torch.inf
    q[2] = 0
    q[3, 2] = 1e-30
    q[4, 0, 7] = -0.0
    turns, axis = _table(gen, parts, 1)
    positions = torch.arange(6)[None] * 7
    table = RotaryAxes(turns.to(dev), axis.to(dev), parts)
    w = _weights(gen, (32, 32))
    got = rotary(q.to(dev), None, positions.to(dev), table, q_norm=HeadNorm(*(x.to(dev) for x in w)))[0].cpu()
    bad = torch.zeros((6, 3, 64), dtype=torch.bool)
    bad[0, 1] = bad[1, 0] = True                                   # (their parts, and what is turned with them)
    keep = ~bad
    want, most = ho.head(q, positions, turns, axis, parts, weights=w)
    assert bool(((got.double() - want).abs() <= most)[keep].all())
    assert bool(torch.isnan(got[0, 1, :32]).any()) and bool(torch.isnan(got[1, 0, 63:]).all()) and not bool(torch.isnan(got[2]).any())
    assert not bool(torch.isnan(got[0, [0, 2]]).any())
    # without a norm, what is not turned is copied bit by bit
    half = RotaryAxes(turns[:8].to(dev).contiguous(), axis[:8].to(dev), (16,))
    copied = rotary(q.to(dev), None, positions.to(dev), half)[0].cpu()
    assert torch.equal(copied[..., 16:].view(torch.int16)[~torch.isnan(q[..., 16:])], q[..., 16:].view(torch.int16)[~torch.isnan(q[..., 16:])])


@pytest.mark.parametrize("quant", [ops.Q8_0, ops.BF16])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,parts,norm,page", [(1, 32, 8, 128, (64, 32, 32), (64, 64), 16), (65, 32, 8, 128, (128,), (128,), 64), (33, 4, 2, 96, (48, 24, 24), (48, 48), 32),
                                                                      (7, 5, 1, 32, (18, 14), (32,), 16), (130, 8, 1, 256, (128, 64, 64), (256,), 128), (40, 3, 3, 64, (64,), (), 16)])
def test_into_the_cache(dev, quant, tokens, q_heads, kv_heads, dim, parts, norm, page):
    gen = torch.Generator().manual_seed(tokens)
    qkv = _values(gen, tokens, q_heads + 2 * kv_heads, dim).to(dev)
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], 1)
    turns, axis = _table(gen, parts, 3)
    table, positions = RotaryAxes(turns.to(dev), axis.to(dev), parts), torch.randint(0, 999, (3, tokens), generator=gen).to(dev)
    norms = dict(q_norm=HeadNorm(*(w.to(dev) for w in _weights(gen, norm))), k_norm=HeadNorm(*(w.to(dev) for w in _weights(gen, norm)))) if norm else {}
    pages = -(-tokens // page) + 2
    cache = PagedKVCache.empty(pages, kv_heads, page, dim, quant, dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(3)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(dev)
    if tokens > 5:
        slots[3], slots[4] = -1, pages * page
    before = [t.clone() for t in (cache.k, cache.v)]
    got = cache.write_rotary(q, k, v, positions, table, slots, **norms)
    want_q, want_k = rotary(q, k, positions, table, **norms)
    assert torch.equal(got, want_q)
    # the same as the turned keys written on their own
    other = PagedKVCache(*(t.clone().fill_(3) if t is not None else None for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    other.write(want_k, v, slots)
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(cache, name) is not None:
            assert torch.equal(getattr(cache, name), getattr(other, name)), name
    untouched = torch.ones(pages * page, dtype=torch.bool, device=dev)
    untouched[slots[(slots >= 0) & (slots < pages * page)]] = False
    for t, b in zip((cache.k, cache.v), before):
        assert torch.equal(t.transpose(1, 2).flatten(0, 1)[untouched], b.transpose(1, 2).flatten(0, 1)[untouched])
    if quant == ops.Q8_0:
        _, _, held = ao.quantised(want_k.cpu()[:1])
        assert torch.equal(cache.read(slots[:1])[0].cpu(), held.to(torch.bfloat16))
    # in place: only the queries
    copy = qkv.clone()
    cache.write_rotary(copy[:, :q_heads], copy[:, q_heads:q_heads + kv_heads], copy[:, q_heads + kv_heads:], positions, table, slots, inplace=True, **norms)
    assert torch.equal(copy[:, :q_heads], got) and torch.equal(copy[:, q_heads:], qkv[:, q_heads:])


@pytest.mark.parametrize("tokens", [1023, 1024, 2049, 5003])
@pytest.mark.parametrize("q_heads,k_heads,dim,parts,norm", [(6, 2, 64, (32, 16, 16), (32, 32)), (40, 0, 32, (32,), ()), (2, 1, 80, (36,), (80,))])
def test_many_tokens(dev, tokens, q_heads, k_heads, dim, parts, norm):
    """Several tokens a workgroup, the last one's fewer."""
    gen = torch.Generator().manual_seed(tokens)
    q, k = _values(gen, tokens, q_heads, dim), _values(gen, tokens, k_heads, dim)
    turns, axis = _table(gen, parts, 2)
    positions, weights = torch.randint(0, 5000, (2, tokens), generator=gen), _weights(gen, norm)
    table = RotaryAxes(turns.to(dev), axis.to(dev), parts)
    norms = dict.fromkeys(("q_norm", "k_norm"), HeadNorm(*(w.to(dev) for w in weights))) if norm else {}
    q2, k2 = rotary(q.to(dev), k.to(dev), positions.to(dev), table, **norms)
    for got, x in ((q2, q), (k2, k)):
        if x.numel():
            _close(got, *ho.head(x, positions, turns, axis, parts, weights=weights, eps=1e-6))
    if k_heads and dim % 32 == 0:
        cache, slots = PagedKVCache.empty(-(-tokens // 64), k_heads, 64, dim, ops.BF16, dev), torch.randperm(tokens, generator=gen).to(dev)
        assert torch.equal(cache.write_rotary(q.to(dev), k.to(dev), k.to(dev), positions.to(dev), table, slots, **norms), q2)
        assert torch.equal(cache.read(slots)[0], k2) and torch.equal(cache.read(slots)[1].cpu(), k)


def test_copies_have_tensors_of_their_own(dev):
    gen = torch.Generator().manual_seed(9)
    q, at = _values(gen, 3, 2, 64).to(dev), torch.randint(0, 99, (2, 3), generator=gen).to(dev)
    axes, norm = RotaryAxes.for_model([(32, 0, 1e4), (32, 1, 1e4)], device=dev), HeadNorm(*(w.to(dev) for w in _weights(gen, (32, 32))), eps=1e-4)
    want = rotary(q, None, at, axes, q_norm=norm)[0]
    copies = [(copy.copy(axes), copy.copy(norm)), copy.deepcopy((axes, norm)), pickle.loads(pickle.dumps((axes, norm)))]
    assert copies[0][1].weights[0] is norm.weights[0]
    for t in (axes.turns, axes.axis, *norm.weights):
        t.zero_()
    assert not torch.equal(rotary(q, None, at, copies[0][0], q_norm=copies[0][1])[0], want)
    for a, n in copies[1:]:
        assert torch.equal(rotary(q, None, at, a, q_norm=n)[0], want)


def test_captured_and_on_another_stream(dev):
    gen = torch.Generator().manual_seed(6)
    qkv = _values(gen, 24, 48, 128).to(dev)
    q, k, v = qkv.split([32, 8, 8], 1)
    table = RotaryAxes.for_model([(64, 0, 5e6), (32, 1, 1e4), (32, 2, 1e4)], device=dev)
    norms = dict(q_norm=HeadNorm(*(w.to(dev) for w in _weights(gen, (64, 64)))), k_norm=HeadNorm(*(w.to(dev) for w in _weights(gen, (64, 64)))))
    positions, slots = torch.randint(0, 999, (3, 24), generator=gen).to(dev), torch.arange(24, device=dev)
    cache = PagedKVCache.empty(4, 8, 16, 128, ops.Q8_0, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write_rotary(q, k, v, positions, table, slots, **norms)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.write_rotary(q, k, v, positions, table, slots, **norms)
    for step in range(4):
        qkv.copy_(_values(gen, 24, 48, 128))
        positions.copy_(torch.randint(0, 9999, (3, 24), generator=gen))
        slots.copy_(torch.randperm(64, generator=gen)[:24])
        graph.replay()
        got = out.clone(), cache.read(slots)
        torch.cuda.synchronize()
        other = PagedKVCache.empty(4, 8, 16, 128, ops.Q8_0, dev)
        want = other.write_rotary(q, k, v, positions, table, slots, **norms)
        assert torch.equal(got[0], want) and all(torch.equal(a, b) for a, b in zip(got[1], other.read(slots))), step


def test_weights_are_read_at_every_call(dev):
    gen = torch.Generator().manual_seed(7)
    q, w = _values(gen, 3, 2, 64).to(dev), torch.ones(64, device=dev)
    table, at = RotaryTable.for_model(64, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    norm = HeadNorm(w)
    one = rotary(q, None, at, table, q_norm=norm)[0]
    w.mul_(2)
    assert torch.equal(rotary(q, None, at, table, q_norm=norm)[0], one * 2)
    p = torch.nn.Parameter(torch.ones(64, device=dev))
    with pytest.raises(ops.SnGgufError, match="requires a gradient"):
        HeadNorm(p)
    with torch.no_grad():
        norm = HeadNorm(p)
    p.data = torch.zeros(64, device=dev)
    torch.cuda.empty_cache()
    assert torch.equal(rotary(q, None, at, table, q_norm=norm)[0], one)


def test_what_does_not_go_together(dev):
    gen = torch.Generator().manual_seed(8)
    q, k = _values(gen, 4, 2, 64).to(dev), _values(gen, 4, 1, 64).to(dev)
    table, axes = RotaryTable.for_model(64, device=dev), RotaryAxes.for_model([(32, 0, 1e4), (32, 1, 1e4)], device=dev)
    one, two = torch.arange(4, device=dev), torch.zeros((2, 4), dtype=torch.int64, device=dev)
    norm, short = HeadNorm(torch.ones(64, device=dev)), HeadNorm(torch.ones(32, device=dev))
    cache = PagedKVCache.empty(1, 1, 16, 64, ops.BF16, dev)
    for message, call in (("positions must be", lambda: rotary(q, k, one, axes)), ("positions must be", lambda: rotary(q, k, two, table, q_norm=norm)),
                          ("positions must be", lambda: rotary(q, k, two[:, :3], axes)), ("positions must be", lambda: rotary(q, k, two.int(), axes)),
                          ("a norm of 32 elements", lambda: rotary(q, k, two, axes, q_norm=short)), ("a norm of 32 elements", lambda: cache.write_rotary(q, k, k, two, axes, one, k_norm=short)),
                          ("pairs do not fit", lambda: rotary(q[..., :32], None, two, axes)), ("up to 512", lambda: rotary(torch.zeros((4, 1, 1024), dtype=torch.bfloat16, device=dev), None, two, axes)),
                          ("share no element", lambda: rotary(q[:, :1].expand(4, 2, 64), None, two, axes, inplace=True)),
                          ("of one type", lambda: HeadNorm(torch.ones(32, device=dev), torch.ones(32, dtype=torch.bfloat16, device=dev))),
                          ("multiple of 8", lambda: HeadNorm(torch.ones(12, device=dev))), ("eps is", lambda: HeadNorm(torch.ones(16, device=dev), eps=-1.0)),
                          ("do not hold", lambda: RotaryAxes(table.turns, axes.axis, (32, 30))), ("do not hold", lambda: RotaryAxes(table.turns, axes.axis, (33, 31))),
                          ("do not hold", lambda: RotaryAxes(table.turns, axes.axis, (16, 16, 16, 8, 8))), ("axis must be", lambda: RotaryAxes(table.turns, axes.axis[:3])),
                          ("axis must be", lambda: RotaryAxes(table.turns, axes.axis.long())), ("magnitude", lambda: RotaryAxes(table.turns, axes.axis, magnitude=math.inf))):
        with pytest.raises(ops.SnGgufError, match=message):
            call()
    assert rotary(q[:0], k[:0], two[:, :0], axes, q_norm=norm)[0].shape == (0, 2, 64)
