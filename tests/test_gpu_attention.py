"""Attention of packed prompts and over the paged cache against 64 bits."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, RotaryTable, ops, paged_attention, prompt_attention, rotary

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu


def _values(gen, tokens, heads, dim, wide=False):
    x = torch.randn((tokens, heads, dim), generator=gen)
    if wide:
        x *= 1 + 3 * (torch.rand((heads, dim), generator=gen) > 0.95)
    return x.to(torch.bfloat16)


def _ends(lens, dev):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)


def _close(got, want, most, what=""):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= most)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, worst {float((off / most)[bad].max()):.3g} times the bound, first at {bad.nonzero()[0].tolist()}"


def _prompt(dev, lens_q, lens_k, heads, kv_heads, dim, causal=True, window=0, seed=0, scale=None):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = _values(gen, sum(lens_q), heads, dim), _values(gen, sum(lens_k), kv_heads, dim, True), _values(gen, sum(lens_k), kv_heads, dim)
    got = prompt_attention(q.to(dev), k.to(dev), v.to(dev), _ends(lens_q, dev), _ends(lens_k, dev), causal=causal, window=window, scale=scale)
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        want, most = ao.attention(q[a:a + n], k[b:b + m], v[b:b + m], causal, window, scale)
        _close(got[a:a + n], want, most, f"sequence of {n} over {m}")
        a, b = a + n, b + m


@pytest.mark.parametrize("length", [1, 2, 15, 16, 31, 33, 63, 64, 65, 127, 128, 129, 200, 517])
def test_prompt_lengths(dev, length):
    _prompt(dev, [length], [length], 8, 2, 128, seed=length)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (32, 8), (28, 4), (5, 1), (12, 1), (40, 8), (130, 1)])
def test_prompt_head_layouts(dev, heads, kv_heads):
    _prompt(dev, [70, 1, 37], [70, 1, 37], heads, kv_heads, 64)


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_dims(dev, dim, causal):
    _prompt(dev, [131, 9], [131, 140], 6, 2, dim, causal)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 1000])
def test_prompt_windows(dev, window):
    _prompt(dev, [300, 5], [300, 333], 4, 2, 128, True, window)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_packed_with_empty_sequences_and_rows_that_see_nothing(dev, causal):
    # no queries; no keys; more queries than keys (the first see nothing); fewer
    _prompt(dev, [0, 5, 90, 3, 0], [7, 0, 40, 150, 0], 8, 4, 128, causal)


def test_prompt_few_rows_over_many_keys_are_split(dev):
    for tokens, keys, causal in ((1, 5000, True), (40, 9001, True), (40, 9001, False)):
        assert ops.load_library().sngguf_attention_workspace_bytes(tokens, keys, 1, 8, 2, 128) > 0
        _prompt(dev, [tokens], [keys], 8, 2, 128, causal)
    _prompt(dev, [3, 1, 30], [4000, 1, 700], 8, 2, 128, True, 900)


def test_prompt_large_scores_and_scales(dev):
    _prompt(dev, [200], [200], 4, 2, 128, scale=5.0)
    _prompt(dev, [200], [200], 4, 2, 128, scale=1e-6)


def test_prompt_views_of_a_stacked_projection(dev):
    gen = torch.Generator().manual_seed(5)
    qkv = torch.cat([_values(gen, 150, 8, 128), _values(gen, 150, 2, 128), _values(gen, 150, 2, 128)], 1)
    q, k, v = qkv.to(dev).split([8, 2, 2], 1)
    got = prompt_attention(q, k, v, _ends([150], dev))
    want, most = ao.attention(*qkv.split([8, 2, 2], 1))
    _close(got, want, most)
    # heads ahead of tokens, rows that start anywhere, elements apart
    flipped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*flipped, _ends([150], dev)), got)
    odd = [torch.empty((150 * x.shape[1] * 128 + 1,), dtype=torch.bfloat16, device=dev)[1:].view(150, x.shape[1], 128).copy_(x) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*odd, _ends([150], dev)), got)
    apart = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*apart, _ends([150], dev)), got)
    # an output with rows of its own layout
    room = torch.full((150, 12, 128), 7.0, dtype=torch.bfloat16, device=dev)
    prompt_attention(q, k, v, _ends([150], dev), out=room[:, 2:10])
    assert torch.equal(room[:, 2:10], got) and bool((room[:, :2] == 7).all()) and bool((room[:, 10:] == 7).all())


def test_prompt_rows_behind_the_last_sequence_are_left_and_other_sequences_stay_apart(dev):
    gen = torch.Generator().manual_seed(6)
    q, k, v = (_values(gen, 200, h, 128).to(dev) for h in (4, 2, 2))
    ends = torch.tensor([0, 70, 150], dtype=torch.int32, device=dev)
    clean = prompt_attention(q, k, v, ends)
    for name in ("nan", "inf"):
        k2, v2 = k.clone(), v.clone()
        k2[70:] = float(name)
        v2[70:] = float(name)
        out = torch.full_like(q, 3.0)
        prompt_attention(q, k2, v2, ends, out=out)
        assert torch.equal(out[:70], clean[:70]) and bool((out[150:] == 3).all())
        k2, v2 = k.clone(), v.clone()
        k2[:70] = float(name)
        v2[150:] = float(name)
        assert torch.equal(prompt_attention(q, k2, v2, ends)[70:150], clean[70:150])


def test_prompt_lengths_that_are_none_stay_within_the_tensors(dev):
    gen = torch.Generator().manual_seed(7)
    q, k, v = (_values(gen, 50, h, 64).to(dev) for h in (4, 2, 2))
    for ends in ([0, 9000], [-5, 50], [50, 0], [40, 60, -1, 10]):
        out = prompt_attention(q, k, v, torch.tensor(ends, dtype=torch.int32, device=dev))
        assert out.shape == q.shape
    torch.cuda.synchronize()


# ---- paged --------------------------------------------------------------------------------------------------------------


def _paged(dev, new, lens, heads, kv_heads, dim, page, qt, window=0, seed=0, max_new=None, ends=True, poison=True, spare=3, scale=None):
    gen = torch.Generator().manual_seed(seed)
    count = [-(-n // page) for n in lens]
    pages = sum(count) + spare
    order = torch.randperm(pages, generator=gen)
    width = max(max(count), 1) + 1
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)      # numbers that are no pages behind the last one
    cache = PagedKVCache.empty(pages, kv_heads, page, dim, qt, dev)
    if poison:
        # what was never written may be anything
        for t in (cache.k, cache.v):
            t.fill_(-128 if qt == ops.Q8_0 else float("nan"))
        for t in (cache.k_scale, cache.v_scale):
            if t is not None:
                t.fill_(float("nan"))
    ks, vs, at = [], [], 0
    for i, n in enumerate(lens):
        table[i, :count[i]] = order[at:at + count[i]].int()
        at += count[i]
        k, v = _values(gen, n, kv_heads, dim, True), _values(gen, n, kv_heads, dim)
        t = torch.arange(n)
        slots = table[i].long()[t // page] * page + t % page
        cache.write(k.to(dev), v.to(dev), slots.to(dev))
        if qt == ops.Q8_0:
            k, v = ao.quantised(k)[2], ao.quantised(v)[2]
        ks.append(k)
        vs.append(v)
    q = _values(gen, sum(new), heads, dim)
    got = paged_attention(q.to(dev), cache, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), _ends(new, dev) if ends else None,
                          max_new=max(new) if max_new is None else max_new, window=window, scale=scale)
    a = 0
    for n, k, v in zip(new, ks, vs):
        want, most = ao.attention(q[a:a + n], k, v, True, window, scale, torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
        _close(got[a:a + n], want, most, f"{n} new of {len(k)}")
        a += n
    return got


BOTH = pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])


@BOTH
@pytest.mark.parametrize("length", [1, 2, 7, 8, 9, 31, 32, 33, 127, 128, 129, 255, 256, 257, 3001])
def test_single_token_lengths(dev, qt, length):
    _paged(dev, [1], [length], 8, 2, 128, 16, qt, seed=length, ends=False)


@BOTH
@pytest.mark.parametrize("page", [16, 32, 64, 128, 4096])
def test_single_tokens_of_ragged_sequences(dev, qt, page):
    _paged(dev, [1] * 7, [1, 300, 17, 2000, 64, 129, 1111], 32, 8, 128, page, qt)


@BOTH
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_paged_dims(dev, qt, dim, new):
    _paged(dev, [new, 1], [333, 60], 6, 2, dim, 32, qt)


@BOTH
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (16, 1), (17, 1), (28, 4), (40, 1), (70, 1)])
@pytest.mark.parametrize("new", [1, 3])
def test_paged_head_layouts(dev, qt, heads, kv_heads, new):
    _paged(dev, [new, new], [100, 290], heads, kv_heads, 64, 16, qt)


@BOTH
@pytest.mark.parametrize("new", [2, 4, 5, 8, 9, 16, 17, 33, 100, 257])
def test_chunk_sizes(dev, qt, new):
    _paged(dev, [new], [new + 190], 8, 2, 128, 16, qt, seed=new)
    _paged(dev, [new], [new], 8, 2, 128, 64, qt, seed=new)


@BOTH
@pytest.mark.parametrize("max_new", [0, 1, 300, 1000])
def test_chunks_beside_single_tokens(dev, qt, max_new):
    """Which kernels run follows what the caller knows; what they compute does not."""
    _paged(dev, [1, 300, 0, 4, 1, 17], [900, 1300, 50, 4, 1, 100], 8, 2, 128, 32, qt, max_new=max_new)


@BOTH
@pytest.mark.parametrize("window", [1, 31, 32, 100, 5000])
def test_paged_windows(dev, qt, window):
    _paged(dev, [1, 1, 70], [700, 20, 800], 8, 2, 128, 16, qt, window=window)
    _paged(dev, [1], [3000], 8, 2, 128, 16, qt, window=window, ends=False)


@BOTH
def test_rows_that_see_nothing_are_zero(dev, qt):
    got = _paged(dev, [1, 5, 3], [0, 2, 9], 8, 2, 128, 16, qt)
    assert bool((got[0] == 0).all()) and bool((got[1:4] == 0).all()) and bool((got[4:] != 0).any())
    got = _paged(dev, [200, 1], [20, 0], 8, 2, 128, 16, qt)
    assert bool((got[:180] == 0).all()) and bool((got[200:] == 0).all())


@BOTH
def test_long_context_split_over_workgroups(dev, qt):
    _paged(dev, [1], [20011], 8, 2, 128, 64, qt, ends=False)
    _paged(dev, [50, 1], [9000, 4000], 8, 2, 128, 64, qt)


def test_widest_queries_and_values_of_an_8_bit_cache(dev):
    """Queries and scales whose products would leave fp16, and a cache at the ends of what it can hold."""
    gen = torch.Generator().manual_seed(8)
    for q_size, k_size, v_size in ((3e4, 1e-6, 60000.0), (1e-30, 60000.0, 1e-7), (1e10, 1e-7, 1.0)):
        q = (_values(gen, 2, 4, 64).double() * q_size).to(torch.bfloat16)
        k, v = ((_values(gen, 90, 2, 64).clamp(-1, 1).double() * s).to(torch.bfloat16) for s in (k_size, v_size))
        cache = PagedKVCache.empty(6, 2, 16, 64, ops.Q8_0, dev)
        cache.write(k.to(dev), v.to(dev), torch.arange(90, device=dev))
        got = paged_attention(q[:1].to(dev), cache, torch.arange(6, dtype=torch.int32, device=dev)[None], torch.tensor([90], dtype=torch.int32, device=dev))
        want, most = ao.attention(q[:1], ao.quantised(k)[2], ao.quantised(v)[2], operand=torch.float16)
        # values below fp16's normal numbers (2^-14) are rounded by half of 2^-24
        _close(got, want, most + 2.0 ** -25)


def test_bad_pages_and_lengths_stay_within_the_cache(dev):
    gen = torch.Generator().manual_seed(9)
    for qt in (ops.Q8_0, ops.BF16):
        cache = PagedKVCache.empty(4, 2, 16, 64, qt, dev)
        cache.write(_values(gen, 64, 2, 64).to(dev), _values(gen, 64, 2, 64).to(dev), torch.arange(64, device=dev))
        for new in (1, 60):
            q = _values(gen, 2 * new, 4, 64).to(dev)
            table = torch.tensor([[-1, 99, 2 ** 31 - 1, -2 ** 31], [3, 2, 1, 0]], dtype=torch.int32, device=dev)
            out = paged_attention(q, cache, table, torch.tensor([5000, 64], dtype=torch.int32, device=dev), _ends([new, new], dev))
            good = paged_attention(q, cache, table[1:].contiguous(), torch.tensor([64], dtype=torch.int32, device=dev),
                                   torch.tensor([new, 2 * new], dtype=torch.int32, device=dev))
            assert bool(torch.isfinite(out.float()).all()) and torch.allclose(out[new:].float(), good[new:].float(), atol=0.05)
            # nothing of a sequence with a negative length
            out = paged_attention(q, cache, table, torch.tensor([-3, 64], dtype=torch.int32, device=dev), _ends([new, new], dev))
            assert bool((out[:new] == 0).all())


@BOTH
def test_more_sequences_than_a_wavefront_has_lanes(dev, qt):
    gen = torch.Generator().manual_seed(10)
    lens = torch.randint(0, 90, (150,), generator=gen).tolist()
    new = [min(n, 1 + 40 * (i % 50 == 3)) for i, n in enumerate(lens)]
    _paged(dev, new, lens, 4, 2, 64, 16, qt)
    _paged(dev, [1] * 150, [max(n, 1) for n in lens], 4, 2, 64, 16, qt, ends=False)


def test_calls_that_are_refused(dev):
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device=dev)
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=dev)
    ends = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    cache = PagedKVCache.empty(4, 2, 16, 64, device=dev)
    table = torch.zeros((1, 4), dtype=torch.int32, device=dev)
    lens = torch.tensor([4], dtype=torch.int32, device=dev)
    slots = torch.arange(4, device=dev)
    refused = [
        lambda: prompt_attention(q.half(), k, k, ends), lambda: prompt_attention(q[0], k, k, ends), lambda: prompt_attention(q, k, k[:3], ends),
        lambda: prompt_attention(q[:, :3], k, k, ends), lambda: prompt_attention(q, k, k, ends.long()), lambda: prompt_attention(q, k, k, ends, ends[:1]),
        lambda: prompt_attention(q, k, k, ends, window=3, causal=False), lambda: prompt_attention(q, k, k, ends, window=-1), lambda: prompt_attention(q, k, k, ends[:0]),
        lambda: prompt_attention(q, k, k, ends, scale=0.0), lambda: prompt_attention(q, k, k, ends.cpu()), lambda: prompt_attention(q, k, k, ends, out=q.float()),
        lambda: prompt_attention(q, k, k, ends, out=torch.empty((4, 4, 128), dtype=q.dtype, device=dev)[..., ::2]),
        lambda: prompt_attention(q.clone().requires_grad_(), k, k, ends),
        lambda: paged_attention(q, cache, table, lens), lambda: paged_attention(q, cache, table.long(), lens, ends), lambda: paged_attention(q, cache, table[0], lens, ends),
        lambda: paged_attention(q[:, :3], cache, table, lens, ends), lambda: paged_attention(q[..., :32], cache, table, lens, ends),
        lambda: paged_attention(q, cache, table, lens.long(), ends), lambda: paged_attention(q, cache, table, lens, ends, max_new=-1),
        lambda: paged_attention(q, cache, table.cpu(), lens, ends), lambda: paged_attention(q, cache, table.expand(2, 4), lens, ends),
        lambda: cache.write(k, k[:3], slots), lambda: cache.write(q, q, slots), lambda: cache.write(k, k, slots.int()), lambda: cache.write(k, k, slots[:3]),
        lambda: cache.read(slots.int()), lambda: cache.read(slots.cpu()), lambda: PagedKVCache(cache.k, cache.v), lambda: PagedKVCache(cache.k, cache.v, cache.k_scale),
        lambda: PagedKVCache(cache.k[..., :40], cache.v[..., :40]), lambda: PagedKVCache.empty(4, 2, 16, 64, ops.Q4_0, dev),
        lambda: PagedKVCache.empty(4, 2, 24, 64, ops.BF16, dev), lambda: PagedKVCache.empty(4, 2, 16, 48, ops.BF16, dev),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ops.SnGgufError):
            call()
            pytest.fail(f"call {i} was taken")


def test_lengths_that_are_none_where_keys_are_split(dev):
    gen = torch.Generator().manual_seed(12)
    q, k, v = _values(gen, 30, 4, 64).to(dev), _values(gen, 6000, 2, 64).to(dev), _values(gen, 6000, 2, 64).to(dev)
    for n in (1, 40):
        ends_q, ends_k = torch.tensor([0, 30] * n, dtype=torch.int32, device=dev), torch.tensor([0, 6000] * n, dtype=torch.int32, device=dev)
        assert prompt_attention(q, k, v, ends_q, ends_k).shape == q.shape
    cache = PagedKVCache.empty(8, 2, 64, 64, ops.Q8_0, dev)
    cache.write(k[:512], v[:512], torch.arange(512, device=dev))
    table = torch.arange(8, dtype=torch.int32, device=dev).repeat(80, 8).contiguous()
    ends = torch.tensor([0, 30] * 40 + [0], dtype=torch.int32, device=dev)
    for max_new in (0, 1, 30):
        assert paged_attention(q, cache, table, torch.full((80,), 4096, dtype=torch.int32, device=dev), ends, max_new=max_new).shape == q.shape
    torch.cuda.synchronize()


def test_no_keys_and_no_queries(dev):
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=dev)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=dev)
    ends = torch.tensor([0, 1, 3], dtype=torch.int32, device=dev)
    assert bool((prompt_attention(q, none, none, ends, torch.zeros(3, dtype=torch.int32, device=dev)) == 0).all())
    assert prompt_attention(q[:0], none, none, torch.zeros(3, dtype=torch.int32, device=dev)).shape == (0, 4, 64)
    assert prompt_attention(q, none, none, torch.zeros(1, dtype=torch.int32, device=dev)).shape == q.shape
    cache = PagedKVCache.empty(2, 2, 16, 64, ops.BF16, dev)
    lens = torch.zeros(3, dtype=torch.int32, device=dev)
    assert bool((paged_attention(q, cache, torch.zeros((3, 0), dtype=torch.int32, device=dev), lens) == 0).all())
    assert paged_attention(q[:0], cache, torch.zeros((0, 4), dtype=torch.int32, device=dev), lens[:0]).shape == (0, 4, 64)


def test_paged_rows_behind_the_last_sequence_are_left(dev):
    gen = torch.Generator().manual_seed(13)
    for qt in (ops.Q8_0, ops.BF16):
        cache = PagedKVCache.empty(4, 2, 16, 64, qt, dev)
        cache.write(_values(gen, 64, 2, 64).to(dev), _values(gen, 64, 2, 64).to(dev), torch.arange(64, device=dev))
        table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
        lens = torch.tensor([20, 32], dtype=torch.int32, device=dev)
        for new in (1, 18):
            q = _values(gen, 2 * new + 5, 4, 64).to(dev)
            out = torch.full_like(q, 9.0)
            paged_attention(q, cache, table, lens, torch.tensor([0, new, 2 * new], dtype=torch.int32, device=dev), out=out)
            assert bool((out[2 * new:] == 9).all()) and not bool((out[:2 * new] == 9).any(1).any(1).all())


@BOTH
def test_offsets_past_32_bits(dev, qt):
    """A cache whose last pages lie behind 2^32 bytes (8 bits) or 2^33 (bf16) of each half."""
    pages, page, heads, dim = 2 ** 17 + 3, 64, 4, 128
    cache = PagedKVCache.empty(pages, heads, page, dim, qt, dev)
    gen = torch.Generator().manual_seed(14)
    k, v, q = _values(gen, 190, heads, dim), _values(gen, 190, heads, dim), _values(gen, 41, 8, dim)
    table = torch.tensor([[pages - 1, 0, pages - 3, 7]], dtype=torch.int32)
    t = torch.arange(190)
    slots = (table[0].long()[t // page] * page + t % page).to(dev)
    cache.write(k.to(dev), v.to(dev), slots)
    got = cache.read(slots)
    held = [ao.quantised(x)[2] if qt == ops.Q8_0 else x.double() for x in (k, v)]
    assert all(torch.equal(a.double().cpu(), b.float().to(torch.bfloat16).double()) for a, b in zip(got, held))
    for new in (1, 41):
        out = paged_attention(q[:new].to(dev), cache, table.to(dev), torch.tensor([190], dtype=torch.int32, device=dev), torch.tensor([0, new], dtype=torch.int32, device=dev))
        want, most = ao.attention(q[:new], *held, operand=torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
        _close(out, want, most)


def test_long_strides_of_packed_keys(dev):
    """Keys far apart: the last lies behind 2^32 bytes."""
    apart = 2 ** 24
    room = torch.zeros((200 * apart,), dtype=torch.bfloat16, device=dev)
    gen = torch.Generator().manual_seed(15)
    q, k, v = _values(gen, 200, 2, 64), _values(gen, 200, 1, 64), _values(gen, 200, 1, 64)
    kd = room.as_strided((200, 1, 64), (apart, 64, 1)).copy_(k)
    vd = room.as_strided((200, 1, 64), (apart, 64, 1), 128).copy_(v)
    got = prompt_attention(q.to(dev), kd, vd, _ends([200], dev))
    want, most = ao.attention(q, k, v)
    _close(got, want, most)


# ---- together, captured, on other streams ---------------------------------------------------------------------------------


def _step(s, cache, table_of_angles):
    from sensenova_u1_amd import rotary

    q = cache.write_rotary(s["q"], s["k"], s["v"], s["positions"], table_of_angles, s["slots"])
    out = paged_attention(q, cache, s["pages"], s["lens"], s["ends"], max_new=s["max_new"])
    q2, k2 = rotary(s["q"], s["k"], s["positions"], table_of_angles)
    own = prompt_attention(q2, k2, s["v"], s["ends"])
    return out, own, cache.read(s["slots"])


@BOTH
@pytest.mark.parametrize("new,max_new", [([1] * 5, 1), ([1, 40, 1, 300, 7], 0)])
def test_captured_steps_replay_with_new_lengths_pages_and_values(dev, qt, new, max_new):
    """One captured step of a layer, replayed over growing contexts with the program's own work between the replays: every replay is what
    the same calls give outside the graph."""
    from sensenova_u1_amd import RotaryTable

    gen = torch.Generator().manual_seed(16)
    tokens, page, width = sum(new), 16, 160
    angles = RotaryTable.for_model(128, 1e6, device=dev)
    caches = [PagedKVCache.empty(5 * width, 2, page, 128, qt, dev) for _ in range(2)]
    for c in caches:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t.zero_()
    s = {"q": torch.zeros((tokens, 8, 128), dtype=torch.bfloat16, device=dev), "k": torch.zeros((tokens, 2, 128), dtype=torch.bfloat16, device=dev),
         "v": torch.zeros((tokens, 2, 128), dtype=torch.bfloat16, device=dev), "positions": torch.zeros(tokens, dtype=torch.int64, device=dev),
         "slots": torch.zeros(tokens, dtype=torch.int64, device=dev), "pages": torch.zeros((5, width), dtype=torch.int32, device=dev),
         "lens": torch.ones(5, dtype=torch.int32, device=dev), "ends": _ends(new, dev), "max_new": max_new}
    lens = torch.zeros(5, dtype=torch.int64)
    _step(s, caches[0], angles)          # (kernels are loaded)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(s, caches[0], angles)
    for replay in range(4):
        order = torch.randperm(5 * width, generator=gen).view(5, width) if replay == 0 else order
        grown = torch.tensor(new) + (torch.randint(0, 200, (5,), generator=gen) if replay else 0)
        at, pos, slots = 0, [], []
        for i, n in enumerate(new):
            first = int(lens[i] + grown[i]) - n
            p = torch.arange(first, first + n)
            pos.append(p)
            slots.append(order[i][p // page] * page + p % page)
        lens += grown
        for name, value in (("positions", torch.cat(pos)), ("slots", torch.cat(slots)), ("pages", order.int()), ("lens", lens.int()),
                            ("q", _values(gen, tokens, 8, 128)), ("k", _values(gen, tokens, 2, 128)), ("v", _values(gen, tokens, 2, 128))):
            s[name].copy_(value)
        graph.replay()
        eager = _step(s, caches[1], angles)
        torch.cuda.synchronize()
        for a, b in zip((captured[0], captured[1], *captured[2]), (eager[0], eager[1], *eager[2])):
            assert torch.equal(a, b), replay
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v_scale, caches[1].v_scale)):
            assert a is None or torch.equal(a, b)


def test_two_graphs_and_other_streams_do_not_share_scratch(dev):
    """Splits of keys write partial results: of two graphs replayed on two streams, and of eager calls on a third."""
    gen = torch.Generator().manual_seed(17)
    work = []
    for n in (9000, 7000, 5000):
        q, k, v = _values(gen, 4, 8, 128).to(dev), _values(gen, n, 2, 128).to(dev), _values(gen, n, 2, 128).to(dev)
        cache = PagedKVCache.empty(-(-n // 64), 2, 64, 128, ops.Q8_0, dev)
        cache.write(k, v, torch.arange(n, device=dev))
        pages = torch.arange(-(-n // 64), dtype=torch.int32, device=dev)[None]
        args = (q, cache, pages, torch.tensor([n], dtype=torch.int32, device=dev), _ends([4], dev))
        work.append((args, paged_attention(*args), (q, k, v, _ends([4], dev), _ends([n], dev)), prompt_attention(q, k, v, _ends([4], dev), _ends([n], dev))))
    torch.cuda.synchronize()
    graphs = []
    for args, _, packed, _ in work[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = (paged_attention(*args), prompt_attention(*packed))
        graphs.append((g, outs))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    eager = []
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager.append((paged_attention(*work[2][0]), prompt_attention(*work[2][2])))
    torch.cuda.synchronize()
    for (_, outs), (_, a, _, b) in zip(graphs, work):
        assert torch.equal(outs[0], a) and torch.equal(outs[1], b)
    assert all(torch.equal(x, work[2][1]) and torch.equal(y, work[2][3]) for x, y in eager)


def test_results_do_not_change_from_call_to_call(dev):
    gen = torch.Generator().manual_seed(18)
    q, k, v = _values(gen, 700, 8, 128).to(dev), _values(gen, 700, 2, 128, True).to(dev), _values(gen, 700, 2, 128).to(dev)
    first = prompt_attention(q, k, v, _ends([300, 400], dev))
    assert all(torch.equal(prompt_attention(q, k, v, _ends([300, 400], dev)), first) for _ in range(10))


def test_scores_that_rise_from_key_to_key(dev):
    """The maximum is passed again and again, by little and by much: weights, sums and results are set right each time."""
    gen = torch.Generator().manual_seed(19)
    lk = 700
    for rise in (0.05, 0.5, 5.0, -0.5):
        k = (_values(gen, lk, 2, 128).float() * 0.1)
        k[:, :, 0] = torch.arange(lk)[:, None] * rise
        k = k.to(torch.bfloat16)
        q = (_values(gen, lk, 4, 128).float() * 0.1)
        q[:, :, 0] = 8.0
        q, v = q.to(torch.bfloat16), _values(gen, lk, 2, 128)
        got = prompt_attention(q.to(dev), k.to(dev), v.to(dev), _ends([lk], dev))
        want, most = ao.attention(q, k, v)
        _close(got, want, most, f"rise {rise}")
        for qt in (ops.Q8_0, ops.BF16):
            cache = PagedKVCache.empty(44, 2, 16, 128, qt, dev)
            cache.write(k.to(dev), v.to(dev), torch.arange(lk, device=dev))
            kk, vv = [ao.quantised(x)[2] if qt == ops.Q8_0 else x for x in (k, v)]
            for new in (1, 200):
                got = paged_attention(q[-new:].to(dev), cache, torch.arange(44, dtype=torch.int32, device=dev)[None], torch.tensor([lk], dtype=torch.int32, device=dev), _ends([new], dev))
                want, most = ao.attention(q[-new:], kk, vv, operand=torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
                _close(got, want, most, f"rise {rise}, {new} new, type {qt}")


def test_many_small_weights_beside_one_large(dev):
    """30000 keys of weight about 2^-25 of the largest: together a thousandth of the sum, each below fp16's smallest step of it."""
    gen = torch.Generator().manual_seed(20)
    lk = 30000
    k = torch.zeros((lk, 1, 64))
    k[5, 0, 0] = 17.33 / 8.0
    q = torch.zeros((1, 2, 64))
    q[..., 0] = 8.0 * 8.0
    v = torch.ones((lk, 1, 64))
    v[5] = -1.0
    q, k, v = (x.to(torch.bfloat16) for x in (q, k, v))
    for qt in (ops.Q8_0, ops.BF16):
        cache = PagedKVCache.empty(469, 1, 64, 64, qt, dev)
        cache.write(k.to(dev), v.to(dev), torch.arange(lk, device=dev))
        kk, vv = [ao.quantised(x)[2] if qt == ops.Q8_0 else x for x in (k, v)]
        got = paged_attention(q.to(dev), cache, torch.arange(469, dtype=torch.int32, device=dev)[None], torch.tensor([lk], dtype=torch.int32, device=dev))
        want, most = ao.attention(q, kk, vv, operand=torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
        _close(got, want, most)


def test_overlapping_outputs_are_refused(dev):
    x = torch.zeros((8, 6, 64), dtype=torch.bfloat16, device=dev)
    q, k, v = x.split([2, 2, 2], 1)
    ends = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    prompt_attention(q, k, v, ends, out=torch.empty((2, 8, 64), dtype=q.dtype, device=dev).transpose(0, 1))
    cache = PagedKVCache.empty(4, 2, 16, 64, ops.BF16, dev)
    pages, lens = torch.zeros((1, 4), dtype=torch.int32, device=dev), torch.tensor([8], dtype=torch.int32, device=dev)
    turns, positions = RotaryTable.for_model(64, device=dev), torch.arange(8, device=dev)
    wide = torch.zeros((8, 1, 64), dtype=torch.bfloat16, device=dev).expand(8, 2, 64)
    for out in (q, k, v, wide):
        with pytest.raises(ops.SnGgufError):
            prompt_attention(q, k, v, ends, out=out)
    for out in (q, wide):
        with pytest.raises(ops.SnGgufError):
            paged_attention(q, cache, pages, lens, ends, out=out)
    for a, b in ((wide, k), (q, wide), (q, q), (wide, None), (wide.transpose(0, 1)[:1].expand(8, 8, 64), None)):
        with pytest.raises(ops.SnGgufError):
            rotary(a, b, positions, turns, inplace=True)
        rotary(a, b, positions, turns)
    for a, b in ((wide, k), (k, k)):
        with pytest.raises(ops.SnGgufError):
            cache.write_rotary(a, b, v, positions, turns, positions, inplace=True)
    rotary(q, k, positions, turns, inplace=True)


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_many_rows_of_all_dims(dev, dim):
    """Workgroups of 256 rows where the dim has them: with the keys of few tiles split, and without."""
    _prompt(dev, [290], [2100], 4, 2, dim, seed=dim)
    _prompt(dev, [1300], [1300], 32, 32, dim, seed=dim)
    _prompt(dev, [700, 31, 520], [700, 90, 600], 32, 16, dim, False, seed=dim)


@BOTH
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_many_rows_of_all_dims_over_the_cache(dev, qt, dim):
    _paged(dev, [290], [2100], 4, 2, dim, 64, qt, seed=dim)
    _paged(dev, [1300], [1311], 32, 32, dim, 32, qt, seed=dim)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_windows_wider_than_any_sequence(dev, window):
    gen = torch.Generator().manual_seed(11)
    q, k, v = _values(gen, 90, 4, 64).to(dev), _values(gen, 50, 2, 64).to(dev), _values(gen, 50, 2, 64).to(dev)
    for n in (1, 9, 90):
        ends, ends_k = _ends([n], dev), _ends([50], dev)
        assert torch.equal(prompt_attention(q[:n], k, v, ends, ends_k, window=window), prompt_attention(q[:n], k, v, ends, ends_k))
    cache = PagedKVCache.empty(4, 2, 16, 64, ops.BF16, dev)
    cache.write(k, v, torch.arange(50, device=dev))
    pages, lens = torch.arange(4, dtype=torch.int32, device=dev)[None], torch.tensor([50], dtype=torch.int32, device=dev)
    for n in (1, 9, 90):
        assert torch.equal(paged_attention(q[:n], cache, pages, lens, _ends([n], dev), window=window), paged_attention(q[:n], cache, pages, lens, _ends([n], dev)))
    for bad in (dict(window=2 ** 63), dict(window=2 ** 64 + 3), dict(max_new=2 ** 63)):
        with pytest.raises(ops.SnGgufError):
            paged_attention(q[:1], cache, pages, lens, **bad)


@BOTH
def test_without_a_workspace(dev, qt):
    """Through the C entry points: keys are not split then, and a workspace that is too small is as none."""
    lib = ops.load_library()
    gen = torch.Generator().manual_seed(12)
    heads, kv_heads, dim, keys, page = 8, 2, 128, 5000, 64
    k, v = _values(gen, keys, kv_heads, dim, True), _values(gen, keys, kv_heads, dim)
    cache = PagedKVCache.empty(keys // page + 1, kv_heads, page, dim, qt, dev)
    kd, vd = k.to(dev), v.to(dev)
    cache.write(kd, vd, torch.arange(keys, device=dev))
    pages = torch.arange(cache.pages, dtype=torch.int32, device=dev)[None].repeat(2, 1)
    lens = torch.tensor([keys, 900], dtype=torch.int32, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    held = (ao.quantised(k)[2], ao.quantised(v)[2]) if qt == ops.Q8_0 else (k, v)
    for new in (1, 200):
        q = _values(gen, 2 * new, heads, dim)
        qd, ends = q.to(dev), _ends([new, new], dev)
        need = lib.sngguf_paged_attention_workspace_bytes(2 * new, 2, new, pages.shape[1] * page, heads, kv_heads, dim)
        assert need > ws.numel()
        for given, nbytes in ((None, 0), (ws.data_ptr(), ws.numel())):
            out = torch.empty_like(qd)
            assert lib.sngguf_paged_attention(qd.data_ptr(), 2 * new, heads, heads * dim, dim, cache._address, pages.data_ptr(), pages.shape[1], pages.shape[1],
                                              lens.data_ptr(), ends.data_ptr(), 2, new, dim ** -0.5, 0, out.data_ptr(), heads * dim, dim, given, nbytes, stream) == 0
            for i, n in enumerate((keys, 900)):
                want, most = ao.attention(q[i * new:(i + 1) * new], held[0][:n], held[1][:n], True, 0, None, torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
                _close(out[i * new:(i + 1) * new], want, most, f"{new} new of {n}")
        if qt == ops.BF16:
            out = torch.empty_like(qd)
            ends_k = _ends([keys - 900, 900], dev)
            assert lib.sngguf_attention(qd.data_ptr(), 2 * new, heads, heads * dim, dim, kd.data_ptr(), kv_heads * dim, dim, vd.data_ptr(), kv_heads * dim, dim, keys,
                                        kv_heads, dim, ends.data_ptr(), ends_k.data_ptr(), 2, dim ** -0.5, 1, 0, out.data_ptr(), heads * dim, dim, None, 0, stream) == 0
            want, most = ao.attention(q[:new], k[:keys - 900], v[:keys - 900])
            _close(out[:new], want, most)
